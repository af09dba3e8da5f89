// Attention over the pages of the 4-bit KV cache (format in kv4.cuh): one CTA per query and query head, one pass
// over the row's pages with a running maximum and sum.
#include <math.h>

#include "kv4.cuh"

namespace jxb {
namespace {

constexpr int kThreads = 128;

struct AttendArgs {
  jx_kv4_cache c;
  int layer, S, Hq, window;
  float scale;
  const void* q;
  long long q_row, q_tok, q_head;
  void* out;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) kv4_attend_kernel(const AttendArgs a) {
  const jx_kv4_cache& c = a.c;
  __shared__ float qs[256], ps[kPage], red[2];
  const int hd = c.head_dim, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hq = blockIdx.y, head = hq / (a.Hq / c.num_kv_heads);
  const int r = blockIdx.x / a.S, i = blockIdx.x - r * a.S;
  const int cnt = c.counts[r], len = min(c.lengths[r], c.row_pages * kPage);
  T* out = static_cast<T*>(a.out) + ((long long)blockIdx.x * a.Hq + hq) * hd;
  if (cnt > a.S && tid == 0) set_status(c.status, JX_ERR_RANGE);
  const int pos = len - cnt + i;
  if (i >= cnt || pos < 0) {
    for (int d = tid; d < hd; d += kThreads) out[d] = from_f<T>(0.f);
    return;
  }
  const T* q = static_cast<const T*>(a.q) + r * a.q_row + i * a.q_tok + hq * a.q_head;
  for (int d = tid; d < hd; d += kThreads) qs[d] = to_f(q[d]);
  const int from = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  __syncthreads();
  for (int pg = from / kPage; pg <= pos / kPage; ++pg) {
    const int id = c.table[(long long)r * c.row_pages + pg];
    if (id < 0 || id >= c.num_pages) {
      if (tid == 0) set_status(c.status, JX_ERR_RANGE);
      continue;
    }
    const unsigned char* blk = kv4_block(c, a.layer, id, head);
    const bf16* ks = reinterpret_cast<const bf16*>(blk + kv4_scale_offset(hd, 0));
    const bf16* vs = reinterpret_cast<const bf16*>(blk + kv4_scale_offset(hd, 1));
    for (int t = warp; t < kPage; t += kThreads / 32) {
      float s = 0.f;
      for (int b = lane; b < hd / 2; b += 32) {
        const int n = blk[t * (hd / 2) + b];
        const float sc = to_f(ks[t * (hd / 32) + b / 16]);
        s += ((float)((n & 15) - 8) * sc) * qs[2 * b] + ((float)((n >> 4) - 8) * sc) * qs[2 * b + 1];
      }
      for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
      const int key = pg * kPage + t;
      if (lane == 0) ps[t] = key >= from && key <= pos ? s * a.scale : -INFINITY;
    }
    __syncthreads();
    float mx = m;
    for (int t = 0; t < kPage; ++t) mx = fmaxf(mx, ps[t]);
    const float f = m == -INFINITY ? 0.f : expf(m - mx);
    m = mx;
    l *= f, o[0] *= f, o[1] *= f;
    for (int t = 0; t < kPage; ++t) {
      const int key = pg * kPage + t;
      if (key < from || key > pos) continue;
      const float p = expf(ps[t] - m);
      l += p;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = tid + j * kThreads;
        if (d < hd) {
          const int n = blk[kPage * (hd / 2) + t * (hd / 2) + d / 2];
          o[j] += p * ((float)((d & 1 ? n >> 4 : n & 15) - 8) * to_f(vs[t * (hd / 32) + d / 32]));
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int d = tid + j * kThreads;
    if (d < hd) out[d] = from_f<T>(l > 0.f ? o[j] / l : (l != l ? l : 0.f));
  }
}

}  // namespace

long long kv4_attend_workspace(const jx_kv4_cache& c, int S, int Hq, int dtype) { return 16; }

int run_kv4_attend(const jx_kv4_cache& c, int layer, int S, int Hq, const void* q, const long long* qs, void* out,
                   float scale, int window, void* ws, int dtype, cudaStream_t s) {
  AttendArgs a;
  a.c = c, a.layer = layer, a.S = S, a.Hq = Hq, a.window = window, a.scale = scale;
  a.q = q, a.q_row = qs[0], a.q_tok = qs[1], a.q_head = qs[2], a.out = out;
  const dim3 grid(c.num_rows * S, Hq);
  if (dtype == JX_BF16) kv4_attend_kernel<bf16><<<grid, kThreads, 0, s>>>(a);
  else kv4_attend_kernel<float><<<grid, kThreads, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

}  // namespace jxb
