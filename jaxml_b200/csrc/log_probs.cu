// Log probabilities of given tokens, entropy and the top alternatives of logits rows.
//
// With m the row's maximum, z = sum exp(x - m) and w = sum exp(x - m) (x - m):
//   log p(id) = (x[id] - m) - log z,   entropy = log z - w / z.
// One CTA per row; the alternatives are taken one after the other in the order of (value, lowest id).
#include <math.h>

#include "common.cuh"

namespace jxb {
namespace {

constexpr int kThreads = 512;

// Order-preserving integer of a float: -0 equals +0, NaN is above infinity.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* sh, Op op) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = 16; d; d >>= 1) v = op(v, __shfl_xor_sync(~0u, v, d));
  __syncthreads();
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  V r = sh[0];
  for (int i = 1; i < kThreads / 32; ++i) r = op(r, sh[i]);
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) log_probs_kernel(const jx_log_probs_args a) {
  __shared__ float sf[kThreads / 32];
  __shared__ unsigned long long sk[kThreads / 32];
  const int row = blockIdx.x, tid = threadIdx.x, V = a.V;
  const T* x = static_cast<const T*>(a.logits) + (long long)row * a.ld;
  float m = -INFINITY;
  for (int i = tid; i < V; i += kThreads) m = fmaxf(m, to_f(x[i]));
  m = block_reduce(m, sf, [](float p, float q) { return fmaxf(p, q); });
  float z = 0.f, w = 0.f;
  for (int i = tid; i < V; i += kThreads) {
    const float d = to_f(x[i]) - m, e = expf(d);
    z += e;
    if (e != 0.f) w += e * d;
  }
  z = block_reduce(z, sf, [](float p, float q) { return p + q; });
  w = block_reduce(w, sf, [](float p, float q) { return p + q; });
  const float lz = logf(z);
  if (tid == 0) {
    const int id = a.ids[row];
    a.log_probs[row] = id < 0 ? 0.f : id >= V ? __uint_as_float(0x7FC00000u) : (to_f(x[id]) - m) - lz;
    a.entropy[row] = lz - w / z;
  }
  unsigned long long below = ~0ull;
  for (int n = 0; n < a.top_n; ++n) {
    unsigned long long best = 0;
    for (int i = tid; i < V; i += kThreads) {
      const unsigned long long k = ((unsigned long long)order_key(to_f(x[i])) << 32) | (uint32_t)~i;
      if (k < below && k > best) best = k;
    }
    best = block_reduce(best, sk, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
    below = best;
    if (tid == 0) {
      const int id = (int)~(uint32_t)best;
      a.top_ids[(long long)row * a.top_n + n] = id;
      a.top_log_probs[(long long)row * a.top_n + n] = (to_f(x[id]) - m) - lz;
    }
  }
}

}  // namespace

int run_token_log_probs(const jx_log_probs_args& a, cudaStream_t s) {
  if (a.dtype == JX_BF16) log_probs_kernel<bf16><<<a.rows, kThreads, 0, s>>>(a);
  else log_probs_kernel<float><<<a.rows, kThreads, 0, s>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

}  // namespace jxb
