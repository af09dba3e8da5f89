// C ABI of libjxb200: argument checks, layout packing and dispatch to the kernels.
#include <stdio.h>
#include <string.h>

#include "common.cuh"

namespace jxb {
int run_norm(int dtype, const jx_norm_args& p, bool pdl, cudaStream_t stream);
int run_gemv(const bf16* W, const bf16* X, long long Np, long long Kp, int M, const jx_epilogue& e, float* ws,
             long long ws_floats, int* counters, int* status, int grid, bool pdl, cudaStream_t stream);
int gemv_workspace_floats(int grid, int mt);
int run_gemm_k128(const bf16* X, const bf16* W, long long Mp, long long Np, long long Kp, const jx_epilogue& e,
                  int* status, bool pdl, cudaStream_t stream);
int run_gemm_f32(const float* X, long long ldx, const float* W, int M, int N, int K, const jx_epilogue& e, bool pdl,
                 cudaStream_t stream);
int run_qkv_rope_append(int dtype, const jx_qkv_args& p, bool pdl, cudaStream_t stream);
int run_attention_generic(int dtype, const jx_attn_args& p, bool pdl, cudaStream_t stream);
int run_rope_apply(int dtype, const jx_rope_args& p, bool pdl, cudaStream_t stream);
int run_sample(const jx_sample_args& p, bool pdl, cudaStream_t stream);
int run_decode_attention(const jx_dattn_args& a, bool pdl, cudaStream_t stream);
void set_gemv_impl(int impl);
void set_dattn_impl(int impl);
void set_gemm_impl(int impl);
void set_gemm_tile_group(int gm);
int run_prefill_attention(const jx_pattn_args& a, bool pdl, cudaStream_t stream);
void set_pattn_impl(int impl);
long long dattn_workspace_bytes(int B, int Hq, int T, int hd, int n_splits);
int dattn_n_splits(int T, int window);
int run_filter_logits(const jx_filter_args& p, cudaStream_t stream);
int run_sample_finalize(const jx_sample_args& p, const unsigned long long* gathered, int n_shards,
                        cudaStream_t stream);

static thread_local char g_err[512] = "";

int note_cuda(const char* where) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return JX_OK;
  snprintf(g_err, sizeof(g_err), "%s: %s", where, cudaGetErrorString(e));
  return JX_ERR_CUDA;
}

int fail(int code, const char* msg) {
  snprintf(g_err, sizeof(g_err), "%s", msg);
  return code;
}

// ------------------------------------------------------------------------------------------------
// K128 pack / unpack
// ------------------------------------------------------------------------------------------------
template <typename S>
__global__ void pack_k128_kernel(const S* __restrict__ src, long long rows, long long cols, long long ld, int transposed,
                                 bf16* __restrict__ dst, long long rp, long long cp) {
  const long long total = rp * cp;
  for (long long o = blockIdx.x * (long long)blockDim.x + threadIdx.x; o < total; o += (long long)gridDim.x * blockDim.x) {
    // invert k128_offset
    const long long unit = o >> 10, within = o & 1023;
    const long long groups = rp >> 3;
    const long long kchunk = unit / groups, rg = unit - kchunk * groups;
    const long long kcore = within >> 6, r8 = (within >> 3) & 7, k8 = within & 7;
    const long long r = rg * 8 + r8, k = kchunk * 128 + kcore * 8 + k8;
    float v = 0.f;
    if (r < rows && k < cols) v = to_f(transposed ? src[k * ld + r] : src[r * ld + k]);
    dst[o] = __float2bfloat16_rn(v);
  }
}

template <typename D>
__global__ void unpack_k128_kernel(const bf16* __restrict__ src, long long rows, long long cols, long long rp,
                                   D* __restrict__ dst, long long ld) {
  const long long total = rows * cols;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / cols, k = i - r * cols;
    dst[r * ld + k] = from_f<D>(__bfloat162float(src[k128_offset(r, k, rp)]));
  }
}

}  // namespace jxb

using namespace jxb;

extern "C" {

const char* jx_version(void) { return "jxb200 0.1 (sm_100a)"; }
const char* jx_last_error(void) { return g_err; }

int jx_device_sm_count(int* out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return note_cuda("cudaGetDevice");
  if (cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return note_cuda("cudaDeviceGetAttribute");
  return JX_OK;
}

int jx_memset_async(void* ptr, int value, long long bytes, void* stream) {
  if (!ptr || bytes < 0) return fail(JX_ERR_ARG, "jx_memset_async: bad pointer or size");
  if (cudaMemsetAsync(ptr, value, (size_t)bytes, (cudaStream_t)stream) != cudaSuccess) return note_cuda("cudaMemsetAsync");
  return JX_OK;
}

int jx_pack_k128(const void* src, int src_dtype, long long rows, long long cols, long long src_ld, int transposed,
                 void* dst, long long rp, long long cp, void* stream) {
  if (!src || !dst) return fail(JX_ERR_ARG, "jx_pack_k128: null pointer");
  if (rp % 8 || cp % 128 || rows > rp || cols > cp || rows < 0 || cols < 0)
    return fail(JX_ERR_SHAPE, "jx_pack_k128: padded sizes must be multiples of 8 (rows) / 128 (cols) and cover the matrix");
  const long long total = rp * cp;
  const int threads = 256;
  const long long blocks = (total + threads - 1) / threads;
  const int grid = (int)(blocks < 65535 * 16 ? blocks : 65535 * 16);
  cudaStream_t s = (cudaStream_t)stream;
  if (src_dtype == JX_F32)
    pack_k128_kernel<float><<<grid, threads, 0, s>>>((const float*)src, rows, cols, src_ld, transposed, (bf16*)dst, rp, cp);
  else if (src_dtype == JX_BF16)
    pack_k128_kernel<bf16><<<grid, threads, 0, s>>>((const bf16*)src, rows, cols, src_ld, transposed, (bf16*)dst, rp, cp);
  else
    return fail(JX_ERR_DTYPE, "jx_pack_k128: dtype must be JX_F32 or JX_BF16");
  return note_cuda("jx_pack_k128");
}

int jx_unpack_k128(const void* src, long long rows, long long cols, long long rp, void* dst, int dst_dtype,
                   long long dst_ld, void* stream) {
  if (!src || !dst) return fail(JX_ERR_ARG, "jx_unpack_k128: null pointer");
  if (rp % 8 || rows > rp) return fail(JX_ERR_SHAPE, "jx_unpack_k128: bad row padding");
  const long long total = rows * cols;
  if (total == 0) return JX_OK;
  const long long blocks = (total + 255) / 256;
  const int grid = (int)(blocks < 65535 * 16 ? blocks : 65535 * 16);
  cudaStream_t s = (cudaStream_t)stream;
  if (dst_dtype == JX_F32)
    unpack_k128_kernel<float><<<grid, 256, 0, s>>>((const bf16*)src, rows, cols, rp, (float*)dst, dst_ld);
  else if (dst_dtype == JX_BF16)
    unpack_k128_kernel<bf16><<<grid, 256, 0, s>>>((const bf16*)src, rows, cols, rp, (bf16*)dst, dst_ld);
  else
    return fail(JX_ERR_DTYPE, "jx_unpack_k128: dtype must be JX_F32 or JX_BF16");
  return note_cuda("jx_unpack_k128");
}

int jx_norm(const jx_norm_args* args, int dtype, int pdl, void* stream) {
  if (!args || !args->h) return fail(JX_ERR_ARG, "jx_norm: args and h are required");
  if (args->out && args->kind == JX_NORM_NONE) return fail(JX_ERR_ARG, "jx_norm: an output needs a norm kind");
  if ((args->out_rp > 0 || args->out2_rp > 0) && dtype != JX_BF16)
    return fail(JX_ERR_DTYPE, "jx_norm: K128 outputs are bfloat16 only");
  const int rc = run_norm(dtype, *args, pdl != 0, (cudaStream_t)stream);
  if (rc != JX_OK) return rc == JX_ERR_CUDA ? note_cuda("jx_norm") : fail(rc, "jx_norm: unsupported sizes or dtype");
  return JX_OK;
}

int jx_set_decode_linear_impl(int impl) {
  if (impl < 0 || impl > 3)
    return fail(JX_ERR_ARG, "jx_set_decode_linear_impl: 0 (by shape), 1 (mma.sync), 2 (tcgen05), 3 (row split)");
  set_gemv_impl(impl);
  return JX_OK;
}

int jx_linear_decode_workspace(int grid, int M, long long* floats_out) {
  if (!floats_out || M <= 0 || M > 64) return fail(JX_ERR_SHAPE, "jx_linear_decode_workspace: M must be in [1, 64]");
  const int mt = M <= 16 ? 1 : (M <= 32 ? 2 : 4);
  *floats_out = gemv_workspace_floats(grid <= 0 ? 148 : grid, mt);
  return JX_OK;
}

int jx_linear_decode(const void* W, const void* X, long long Np, long long Kp, int M, const jx_epilogue* epi,
                     float* ws, long long ws_floats, int* counters, int* status, int grid, int pdl, void* stream) {
  if (!W || !X || !epi || !ws || !counters) return fail(JX_ERR_ARG, "jx_linear_decode: null pointer");
  const int rc = run_gemv((const bf16*)W, (const bf16*)X, Np, Kp, M, *epi, ws, ws_floats, counters, status, grid,
                          pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_linear_decode");
  if (rc != JX_OK)
    return fail(rc, "jx_linear_decode: bad shape (M<=64, Np%64, Kp%128), alignment, workspace or push fields");
  return JX_OK;
}

int jx_linear_prefill(const void* X, const void* W, long long Mp, long long Np, long long Kp, const jx_epilogue* epi,
                      int* status, int pdl, void* stream) {
  if (!W || !X || !epi) return fail(JX_ERR_ARG, "jx_linear_prefill: null pointer");
  if (epi->kind == JX_EPI_PUSH_F32) return fail(JX_ERR_UNSUPPORTED, "jx_linear_prefill: the push epilogue is decode-only");
  const int rc = run_gemm_k128((const bf16*)X, (const bf16*)W, Mp, Np, Kp, *epi, status, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_linear_prefill");
  if (rc != JX_OK) return fail(rc, "jx_linear_prefill: Mp, Np and Kp must be multiples of 128");
  return JX_OK;
}

int jx_linear_f32(const float* X, long long ldx, const float* W, int M, int N, int K, const jx_epilogue* epi, int pdl,
                  void* stream) {
  if (!X || !W || !epi) return fail(JX_ERR_ARG, "jx_linear_f32: null pointer");
  if (epi->kind == JX_EPI_PUSH_F32) return fail(JX_ERR_UNSUPPORTED, "jx_linear_f32: the push epilogue is decode-only");
  const int rc = run_gemm_f32(X, ldx, W, M, N, K, *epi, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_linear_f32");
  if (rc != JX_OK) return fail(rc, "jx_linear_f32: bad shape");
  return JX_OK;
}

int jx_qkv_rope_append(const jx_qkv_args* args, int dtype, int pdl, void* stream) {
  if (!args || !args->qkv || !args->q_out || !args->k_cache || !args->v_cache || !args->cos || !args->sin)
    return fail(JX_ERR_ARG, "jx_qkv_rope_append: null pointer");
  if (args->decode && !args->pos_id) return fail(JX_ERR_ARG, "jx_qkv_rope_append: decode needs pos_id");
  const int rc = run_qkv_rope_append(dtype, *args, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_qkv_rope_append");
  if (rc != JX_OK) return fail(rc, "jx_qkv_rope_append: unsupported head size / rotary dim / dtype");
  return JX_OK;
}

int jx_rope_apply(const jx_rope_args* args, int dtype, int pdl, void* stream) {
  if (!args || !args->cos || !args->sin || !args->pos || (args->Hq > 0 && (!args->q || !args->q_out)) ||
      (args->Hk > 0 && (!args->k || !args->k_out)))
    return fail(JX_ERR_ARG, "jx_rope_apply: null pointer");
  const int rc = run_rope_apply(dtype, *args, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_rope_apply");
  if (rc != JX_OK) return fail(rc, "jx_rope_apply: unsupported head size / rotary dim / dtype");
  return JX_OK;
}

int jx_attention(const jx_attn_args* args, int dtype, int pdl, void* stream) {
  if (!args || !args->q || !args->k || !args->v || !args->out) return fail(JX_ERR_ARG, "jx_attention: null pointer");
  if (args->out_rp > 0 && dtype != JX_BF16) return fail(JX_ERR_DTYPE, "jx_attention: K128 output is bfloat16 only");
  const int rc = run_attention_generic(dtype, *args, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_attention");
  if (rc != JX_OK) return fail(rc, "jx_attention: unsupported sizes or dtype");
  return JX_OK;
}

int jx_decode_attention_workspace(int B, int Hq, int hd, int T, int window, long long* bytes_out) {
  if (!bytes_out || B <= 0 || Hq <= 0 || hd <= 0 || T <= 0) return fail(JX_ERR_SHAPE, "jx_decode_attention_workspace: bad sizes");
  *bytes_out = dattn_workspace_bytes(B, Hq, T, hd, dattn_n_splits(T, window));
  return JX_OK;
}

int jx_decode_attention(const jx_dattn_args* args, int pdl, void* stream) {
  if (!args || !(args->q || args->qkv) || !args->k_base || !args->v_base || !args->out || !args->ws || !args->counters ||
      !args->len_ptr)
    return fail(JX_ERR_ARG, "jx_decode_attention: null pointer");
  const int rc = run_decode_attention(*args, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_decode_attention");
  if (rc == JX_ERR_UNSUPPORTED) return fail(rc, "jx_decode_attention: the fused RoPE inputs (qkv) need the split form");
  if (rc != JX_OK)
    return fail(rc, "jx_decode_attention: head_dim must be 64/128/256, Hq/Hkv <= 16, out_rp >= B and a multiple "
                    "of 8, workspace large enough, 16-byte aligned q/cache, and with qkv: tables, 0 < rd <= hd "
                    "even, ld_qkv >= (Hq + 2 Hkv) hd and a multiple of 8");
  return JX_OK;
}

int jx_set_prefill_tile_group(int gm) {
  if (gm < 0) return fail(JX_ERR_ARG, "jx_set_prefill_tile_group: gm >= 0");
  set_gemm_tile_group(gm);
  return JX_OK;
}

int jx_set_prefill_linear_impl(int impl) {
  if (impl < 0 || impl > 2)
    return fail(JX_ERR_ARG, "jx_set_prefill_linear_impl: 0 (by shape), 1 (mma.sync), 2 (tcgen05)");
  set_gemm_impl(impl);
  return JX_OK;
}

int jx_set_decode_attention_impl(int impl) {
  if (impl < 0 || impl > 5)
    return fail(JX_ERR_ARG, "jx_set_decode_attention_impl: 0 (by shape), 1 (split), 2 (cluster), 3 (column pv), "
                            "4 (cluster-split), 5 (queue)");
  set_dattn_impl(impl);
  return JX_OK;
}

int jx_set_prefill_attention_impl(int impl) {
  if (impl < 0 || impl > 2)
    return fail(JX_ERR_ARG, "jx_set_prefill_attention_impl: 0 (by shape), 1 (mma.sync), 2 (tcgen05)");
  set_pattn_impl(impl);
  return JX_OK;
}

int jx_prefill_attention(const jx_pattn_args* args, int pdl, void* stream) {
  if (!args || !args->q || !args->k_base || !args->v_base || !args->out || !args->len_ptr)
    return fail(JX_ERR_ARG, "jx_prefill_attention: null pointer");
  const int rc = run_prefill_attention(*args, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_prefill_attention");
  if (rc != JX_OK) return fail(rc, "jx_prefill_attention: head_dim must be 64/128/256, Hq % Hkv == 0, S <= T");
  return JX_OK;
}

int jx_filter_logits(const jx_filter_args* args, void* stream) {
  if (!args || !args->logits || !args->out) return fail(JX_ERR_ARG, "jx_filter_logits: null pointer");
  const int rc = run_filter_logits(*args, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_filter_logits");
  if (rc == JX_ERR_DTYPE) return fail(rc, "jx_filter_logits: logits must be float32 or bfloat16");
  if (rc != JX_OK) return fail(rc, "jx_filter_logits: B <= 8191, 0 < V <= 393216 and V <= each leading dimension");
  return JX_OK;
}

int jx_sample(const jx_sample_args* args, int pdl, void* stream) {
  if (!args || !args->logits || !args->ws || !args->counters) return fail(JX_ERR_ARG, "jx_sample: null pointer");
  if (!args->greedy && (!args->rng || (args->dtype == JX_BF16 && !args->gumbel_tab)))
    return fail(JX_ERR_ARG, "jx_sample: temperature sampling needs rng state and the Gumbel table");
  if (!args->greedy && !(args->temp > 0.f)) return fail(JX_ERR_ARG, "jx_sample: temperature must be positive");
  if (!args->finalize && !args->row_best) return fail(JX_ERR_ARG, "jx_sample: finalize == 0 needs row_best");
  const int rc = run_sample(*args, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_sample");
  if (rc != JX_OK) return fail(rc, "jx_sample: bad sizes or dtype");
  return JX_OK;
}

int jx_sample_finalize(const jx_sample_args* args, const unsigned long long* gathered, int n_shards, void* stream) {
  if (!args || !gathered || n_shards <= 0) return fail(JX_ERR_ARG, "jx_sample_finalize: bad arguments");
  const int rc = run_sample_finalize(*args, gathered, n_shards, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_sample_finalize");
  if (rc != JX_OK) return fail(rc, "jx_sample_finalize: bad sizes");
  return JX_OK;
}

}  // extern "C"

// ------------------------------------------------------------------------------------------------
// tensor-parallel peer memory and all-reduce
// ------------------------------------------------------------------------------------------------
namespace jxb {
long long ar_region_bytes(long long max_floats, int world);
long long ar_data_offset(long long max_floats, int which);
void comm_layout(long long max_floats, int world, long long* out);
int run_allreduce_f32(void* const* bases, int rank, int world, long long max_floats, int which, long long n,
                      float* out, int* status, bool pdl, cudaStream_t s);
}  // namespace jxb

extern "C" {

int jx_comm_alloc(long long bytes, void** ptr_out) {
  if (!ptr_out || bytes <= 0) return fail(JX_ERR_ARG, "jx_comm_alloc: null output or non-positive size");
  void* p = nullptr;
  if (cudaMalloc(&p, (size_t)bytes) != cudaSuccess) return note_cuda("jx_comm_alloc");
  if (cudaMemset(p, 0, (size_t)bytes) != cudaSuccess) {
    cudaFree(p);
    return note_cuda("jx_comm_alloc");
  }
  *ptr_out = p;
  return JX_OK;
}

int jx_comm_free(void* ptr) {
  if (!ptr) return JX_OK;
  return cudaFree(ptr) == cudaSuccess ? JX_OK : note_cuda("jx_comm_free");
}

int jx_ipc_get_handle(const void* ptr, unsigned char* handle_out) {
  if (!ptr || !handle_out) return fail(JX_ERR_ARG, "jx_ipc_get_handle: null pointer");
  cudaIpcMemHandle_t h;
  if (cudaIpcGetMemHandle(&h, const_cast<void*>(ptr)) != cudaSuccess) return note_cuda("jx_ipc_get_handle");
  memcpy(handle_out, &h, sizeof(h));
  return JX_OK;
}

int jx_ipc_open_handle(const unsigned char* handle, void** ptr_out) {
  if (!handle || !ptr_out) return fail(JX_ERR_ARG, "jx_ipc_open_handle: null pointer");
  cudaIpcMemHandle_t h;
  memcpy(&h, handle, sizeof(h));
  void* p = nullptr;
  if (cudaIpcOpenMemHandle(&p, h, cudaIpcMemLazyEnablePeerAccess) != cudaSuccess) return note_cuda("jx_ipc_open_handle");
  *ptr_out = p;
  return JX_OK;
}

int jx_ipc_close_handle(void* ptr) {
  if (!ptr) return JX_OK;
  return cudaIpcCloseMemHandle(ptr) == cudaSuccess ? JX_OK : note_cuda("jx_ipc_close_handle");
}

int jx_comm_layout(long long max_floats, int world, long long* out10) {
  if (max_floats <= 0 || world < 1 || world > 8 || !out10)
    return fail(JX_ERR_ARG, "jx_comm_layout: max_floats > 0, 1 <= world <= 8, non-null output");
  jxb::comm_layout(max_floats, world, out10);
  return JX_OK;
}

int jx_allreduce_f32(void* const* bases, int rank, int world, long long max_floats, int which, long long n,
                     float* out, int* status, int pdl, void* stream) {
  if (!bases) return fail(JX_ERR_ARG, "jx_allreduce_f32: null region table");
  const int rc =
      jxb::run_allreduce_f32(bases, rank, world, max_floats, which, n, out, status, pdl != 0, (cudaStream_t)stream);
  if (rc == JX_ERR_CUDA) return note_cuda("jx_allreduce_f32");
  if (rc != JX_OK)
    return fail(rc, "jx_allreduce_f32: 1 <= world <= 8, 0 <= rank < world, which 0 or 1, n a positive multiple "
                    "of 4 and at most max_floats, every region 256-byte aligned, out 16-byte aligned");
  return JX_OK;
}

}  // extern "C"

// ------------------------------------------------------------------------------------------------
// paged 4-bit KV cache and scoring
// ------------------------------------------------------------------------------------------------
namespace jxb {
int run_kv4_append(const jx_kv4_cache& c, int layer, int S, const void* k, const void* v, const long long* ks,
                   const long long* vs, int dtype, cudaStream_t s);
int run_kv4_read(const jx_kv4_cache& c, int layer, const int* start, int start_add, int n, void* k, void* v, int dtype,
                 cudaStream_t s);
long long kv4_workspace_ints(int rows, int pages);
int run_kv4_extend(const jx_kv4_cache& c, const int* counts, int count, int* ws, cudaStream_t s);
int run_kv4_compact(const jx_kv4_cache& c, int* used, int* ws, cudaStream_t s);
int run_kv4_fork(const jx_kv4_cache& c, const int* parents, cudaStream_t s);
int run_kv4_shorten(const jx_kv4_cache& c, const unsigned char* rows, const int* n, int n_all, cudaStream_t s);
long long kv4_attend_workspace(const jx_kv4_cache& c, int S, int Hq, int dtype);
int run_kv4_attend(const jx_kv4_cache& c, int layer, int S, int Hq, const void* q, const long long* qs, void* out,
                   float scale, int window, void* ws, int dtype, cudaStream_t s);
int run_token_log_probs(const jx_log_probs_args& a, cudaStream_t s);

// The checks every call on a cache makes; a message on failure.
static const char* kv4_bad(const jx_kv4_cache* c, int* code) {
  *code = JX_ERR_ARG;
  if (!c) return "null cache";
  if (!c->pages || !c->table || !c->lengths || !c->counts || !c->refs || !c->status) return "null cache pointer";
  if ((uintptr_t)c->pages & 15) return "pages must be 16-byte aligned";
  *code = JX_ERR_SHAPE;
  if (c->num_layers <= 0 || c->num_pages <= 0 || c->num_rows <= 0 || c->row_pages <= 0 || c->num_kv_heads <= 0)
    return "cache sizes must be positive";
  if (c->num_rows > 8192) return "at most 8192 rows";
  if (c->row_pages > (1 << 24)) return "at most 2^24 pages per row";
  // the pages that all rows ask for are counted in 32 bits
  if ((long long)c->num_rows * c->row_pages > 0x7FFFFFFF) return "the table must have fewer than 2^31 entries";
  if (c->num_pages > (1 << 28) || c->num_kv_heads > 4096) return "at most 2^28 pages and 4096 KV heads";
  if ((long long)c->num_layers * c->num_pages * c->num_kv_heads > 0x7FFFFFFF) return "layers * pages * KV heads must be below 2^31";
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "head_dim must be 64, 128 or 256";
  return nullptr;
}

static int kv4_fail(int code, const char* where, const char* msg) {
  snprintf(g_err, sizeof(g_err), "%s: %s", where, msg);
  return code;
}

// Whether a call's row vector lies in memory that the call changes while it is read.  `whole`: the cache's own lengths or counts,
// from their first entry, are fine (a row's entries are read before they are written).
static bool kv4_in_state(const jx_kv4_cache& c, const void* p, long long bytes, bool whole) {
  if (!p || (whole && (p == c.lengths || p == c.counts))) return false;
  const uintptr_t from = (uintptr_t)p, to = from + bytes;
  auto meets = [&](const void* q, long long n) { return from < (uintptr_t)q + n && (uintptr_t)q < to; };
  return meets(c.table, 4ll * c.num_rows * c.row_pages) || meets(c.lengths, 4ll * c.num_rows) || meets(c.counts, 4ll * c.num_rows) ||
         meets(c.refs, 4ll * c.num_pages) || meets(c.status, 4);
}

static int kv4_done(int rc, const char* where) { return rc == JX_ERR_CUDA ? note_cuda(where) : rc; }
}  // namespace jxb

#define KV4_CHECK(where)                                                   \
  int bad_code;                                                            \
  if (const char* bad_msg = kv4_bad(cache, &bad_code)) return kv4_fail(bad_code, where, bad_msg)

extern "C" {

int jx_kv4_append(const jx_kv4_cache* cache, int layer, int S, const void* k, long long k_row, long long k_tok,
                  long long k_head, const void* v, long long v_row, long long v_tok, long long v_head, int dtype,
                  void* stream) {
  KV4_CHECK("jx_kv4_append");
  if (!k || !v) return fail(JX_ERR_ARG, "jx_kv4_append: null keys or values");
  if (layer < 0 || layer >= cache->num_layers || S <= 0 || S > (1 << 30))
    return fail(JX_ERR_SHAPE, "jx_kv4_append: layer out of range, or S not within [1, 2^30]");
  if (dtype != JX_F32 && dtype != JX_BF16) return fail(JX_ERR_DTYPE, "jx_kv4_append: float32 or bfloat16");
  const uintptr_t size = dtype == JX_BF16 ? 2 : 4;
  if ((uintptr_t)k % size || (uintptr_t)v % size) return fail(JX_ERR_ARG, "jx_kv4_append: misaligned keys or values");
  const long long ks[3] = {k_row, k_tok, k_head}, vs[3] = {v_row, v_tok, v_head};
  return kv4_done(run_kv4_append(*cache, layer, S, k, v, ks, vs, dtype, (cudaStream_t)stream), "jx_kv4_append");
}

int jx_kv4_read(const jx_kv4_cache* cache, int layer, const int* start, int start_add, int n, void* k, void* v, int dtype,
                void* stream) {
  KV4_CHECK("jx_kv4_read");
  if (!k || !v || ((uintptr_t)k & 15) || ((uintptr_t)v & 15))
    return fail(JX_ERR_ARG, "jx_kv4_read: outputs must be 16-byte aligned");
  if (layer < 0 || layer >= cache->num_layers || n <= 0 || n > (1 << 30))
    return fail(JX_ERR_SHAPE, "jx_kv4_read: layer out of range, or n not within [1, 2^30]");
  if (dtype != JX_F32 && dtype != JX_BF16) return fail(JX_ERR_DTYPE, "jx_kv4_read: float32 or bfloat16");
  return kv4_done(run_kv4_read(*cache, layer, start, start_add, n, k, v, dtype, (cudaStream_t)stream), "jx_kv4_read");
}

int jx_kv4_attend_workspace(const jx_kv4_cache* cache, int S, int Hq, int dtype, long long* bytes) {
  KV4_CHECK("jx_kv4_attend_workspace");
  if (!bytes) return fail(JX_ERR_ARG, "jx_kv4_attend_workspace: null output");
  if (S <= 0 || Hq <= 0 || Hq % cache->num_kv_heads)
    return fail(JX_ERR_SHAPE, "jx_kv4_attend_workspace: S >= 1, Hq a multiple of the KV heads");
  *bytes = kv4_attend_workspace(*cache, S, Hq, dtype);
  return JX_OK;
}

int jx_kv4_attend(const jx_kv4_cache* cache, int layer, int S, int Hq, const void* q, long long q_row, long long q_tok,
                  long long q_head, void* out, float scale, int window, void* ws, long long ws_bytes, int dtype,
                  void* stream) {
  KV4_CHECK("jx_kv4_attend");
  if (!q || !out || ((uintptr_t)out & 15) || ((uintptr_t)ws & 15))
    return fail(JX_ERR_ARG, "jx_kv4_attend: null pointer, or out / ws not 16-byte aligned");
  if (layer < 0 || layer >= cache->num_layers || S <= 0 || window < 0)
    return fail(JX_ERR_SHAPE, "jx_kv4_attend: layer out of range, S < 1 or window < 0");
  if (Hq <= 0 || Hq % cache->num_kv_heads || Hq > 65535)
    return fail(JX_ERR_SHAPE, "jx_kv4_attend: Hq must be a multiple of the KV heads, at most 65535");
  if ((long long)cache->num_rows * S > 0x7FFFFFFF / Hq) return fail(JX_ERR_SHAPE, "jx_kv4_attend: rows * S * Hq must be below 2^31");
  if (dtype != JX_F32 && dtype != JX_BF16) return fail(JX_ERR_DTYPE, "jx_kv4_attend: float32 or bfloat16");
  if ((uintptr_t)q % (dtype == JX_BF16 ? 2 : 4)) return fail(JX_ERR_ARG, "jx_kv4_attend: misaligned queries");
  if (!(scale > -1e30f && scale < 1e30f)) return fail(JX_ERR_ARG, "jx_kv4_attend: scale must be finite");
  if ((ws ? ws_bytes : 0) < kv4_attend_workspace(*cache, S, Hq, dtype))
    return fail(JX_ERR_ARG, "jx_kv4_attend: workspace too small");
  const long long qs[3] = {q_row, q_tok, q_head};
  return kv4_done(run_kv4_attend(*cache, layer, S, Hq, q, qs, out, scale, window, ws, dtype, (cudaStream_t)stream),
                  "jx_kv4_attend");
}

int jx_kv4_workspace_ints(const jx_kv4_cache* cache, long long* ints) {
  KV4_CHECK("jx_kv4_workspace_ints");
  if (!ints) return fail(JX_ERR_ARG, "jx_kv4_workspace_ints: null output");
  *ints = kv4_workspace_ints(cache->num_rows, cache->num_pages);
  return JX_OK;
}

int jx_kv4_extend(const jx_kv4_cache* cache, const int* counts, int count, int* ws, long long ws_ints, void* stream) {
  KV4_CHECK("jx_kv4_extend");
  if (!counts && count < 0) return fail(JX_ERR_SHAPE, "jx_kv4_extend: count must not be negative");
  if (!ws || ws_ints < kv4_workspace_ints(cache->num_rows, cache->num_pages))
    return fail(JX_ERR_ARG, "jx_kv4_extend: workspace too small");
  if (kv4_in_state(*cache, counts, 4ll * cache->num_rows, true))
    return fail(JX_ERR_ARG, "jx_kv4_extend: counts must not lie in the cache's own state, but be its lengths or counts");
  return kv4_done(run_kv4_extend(*cache, counts, count, ws, (cudaStream_t)stream), "jx_kv4_extend");
}

int jx_kv4_fork(const jx_kv4_cache* cache, const int* parents, void* stream) {
  KV4_CHECK("jx_kv4_fork");
  if (!parents) return fail(JX_ERR_ARG, "jx_kv4_fork: null parents");
  if (kv4_in_state(*cache, parents, 4ll * cache->num_rows, false))
    return fail(JX_ERR_ARG, "jx_kv4_fork: parents must not lie in the cache's own state");
  return kv4_done(run_kv4_fork(*cache, parents, (cudaStream_t)stream), "jx_kv4_fork");
}

int jx_kv4_rollback(const jx_kv4_cache* cache, const int* n, int n_all, void* stream) {
  KV4_CHECK("jx_kv4_rollback");
  if (!n && n_all < 0) return fail(JX_ERR_SHAPE, "jx_kv4_rollback: n must not be negative");
  if (kv4_in_state(*cache, n, 4ll * cache->num_rows, true))
    return fail(JX_ERR_ARG, "jx_kv4_rollback: n must not lie in the cache's own state, but be its lengths or counts");
  return kv4_done(run_kv4_shorten(*cache, nullptr, n, n_all, (cudaStream_t)stream), "jx_kv4_rollback");
}

int jx_kv4_free(const jx_kv4_cache* cache, const unsigned char* rows, void* stream) {
  KV4_CHECK("jx_kv4_free");
  if (!rows) return fail(JX_ERR_ARG, "jx_kv4_free: null rows");
  if (kv4_in_state(*cache, rows, cache->num_rows, false))
    return fail(JX_ERR_ARG, "jx_kv4_free: rows must not lie in the cache's own state");
  return kv4_done(run_kv4_shorten(*cache, rows, nullptr, 0, (cudaStream_t)stream), "jx_kv4_free");
}

int jx_kv4_compact(const jx_kv4_cache* cache, int* used, int* ws, long long ws_ints, void* stream) {
  KV4_CHECK("jx_kv4_compact");
  if (!used) return fail(JX_ERR_ARG, "jx_kv4_compact: null output");
  if (!ws || ws_ints < kv4_workspace_ints(cache->num_rows, cache->num_pages))
    return fail(JX_ERR_ARG, "jx_kv4_compact: workspace too small");
  return kv4_done(run_kv4_compact(*cache, used, ws, (cudaStream_t)stream), "jx_kv4_compact");
}

int jx_token_log_probs(const jx_log_probs_args* args, void* stream) {
  if (!args || !args->logits || !args->ids || !args->log_probs || !args->entropy)
    return fail(JX_ERR_ARG, "jx_token_log_probs: null pointer");
  if (args->rows <= 0 || args->V <= 0 || (args->rows > 1 && args->ld < args->V))
    return fail(JX_ERR_SHAPE, "jx_token_log_probs: sizes must be positive and rows must not overlap");
  if (args->V > (1 << 30)) return fail(JX_ERR_SHAPE, "jx_token_log_probs: V must be at most 2^30");
  if (args->top_n < 0 || args->top_n > 64 || args->top_n > args->V)
    return fail(JX_ERR_SHAPE, "jx_token_log_probs: 0 <= top_n <= min(64, V)");
  if (args->top_n && (!args->top_log_probs || !args->top_ids))
    return fail(JX_ERR_ARG, "jx_token_log_probs: null pointer for the alternatives");
  if (args->dtype != JX_F32 && args->dtype != JX_BF16) return fail(JX_ERR_DTYPE, "jx_token_log_probs: float32 or bfloat16");
  if ((uintptr_t)args->logits % (args->dtype == JX_BF16 ? 2 : 4)) return fail(JX_ERR_ARG, "jx_token_log_probs: misaligned logits");
  return kv4_done(run_token_log_probs(*args, (cudaStream_t)stream), "jx_token_log_probs");
}

}  // extern "C"
