// Log probabilities of given tokens, entropy and the top alternatives of logits rows.
//
// With m the row's maximum, z = sum exp(x - m) and w = sum exp(x - m) (x - m):
//   log p(id) = (x[id] - m) - log z,   entropy = log z - w / z.
// One reading of the row.  A thread keeps a reference K of its own, in units of log2: u = x log2(e) - K is one fused
// multiply-add, z = sum 2^u and w = sum 2^u u, and both move to the reference of a new maximum when a batch of elements
// brings one.  K is rounded, but it is the same K for every element: the joined reference enters the results in 64 bits, as K
// over the float32 constant that x was multiplied with, once a row.  Rows of magnitude above 2^13 (where a rounded K would be
// far from the maximum in units of u), and rows with NaN or infinity, are read again the careful way: x - m first, which is
// exact near the maximum.  The relative error of all log probabilities of 1024 rows of 128256, and the alternatives', is
// 6.2e-8; elementary float32 operations on x - m give 4.4e-8.
//
// The alternatives come from the maxima of the threads and of their batches.  t, the top_n-th largest of the threads'
// maxima, is a lower bound of every element wanted, and the larger elements lie in batches (whose maxima stay in shared
// memory) of fewer than top_n threads: only those are read again.  Up to an eighth of the threads, t is the top_n-th largest
// of the maxima of groups of 4 threads, a little lower a bound for a sixteenth of the comparisons, and the larger elements lie
// in batches of fewer than 4 top_n threads.  Elements equal to t are taken in the order of their index until top_n are there.
//
// What bounds it is half the reading of the logits, half instructions (73 warp instructions for 8 elements of each lane, 8
// of them exponentials at a quarter of the rate) and the alternatives' trip back to the row's batches at its end.  Few rows
// are split over a cluster of CTAs, whose results meet in the first one's shared memory.  Measured (B200): 1024 rows of
// 128256 bfloat16 logits 51 us (5.2 TB/s) without alternatives, 64 us with 20; 7 rows of 50304 in float32 11 us.
#include <math.h>

#include "common.cuh"

namespace jxb {
namespace {

constexpr int kSlots = 32;        // batch maxima a thread keeps; a batch is 4 vectors times a whole number of rounds
constexpr int kCand = 1024;       // elements above t that fit; more (all in a few batches) take the slow way
constexpr int kMostTop = 64;

__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7FC00000u); }
// Order-preserving integer of a float: -0 equals +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two floats at a time.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// z and w of a set of elements relative to a reference; m: its maximum (NaN where the set has one).
struct Sums {
  double ref;      // natural units, -inf without elements
  float m, z, w;   // w in natural units
};
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
  Sums r;
  r.m = max_nan(a.m, b.m);
  r.ref = fmax(a.ref, b.ref);
  const float da = a.ref == r.ref ? 0.f : fmaxf((float)(a.ref - r.ref), -1e30f);
  const float db = b.ref == r.ref ? 0.f : fmaxf((float)(b.ref - r.ref), -1e30f);
  const float fa = exp2_f(da * 1.4426950408889634f), fb = exp2_f(db * 1.4426950408889634f);
  r.z = a.z * fa + b.z * fb;
  r.w = fa * (a.w + a.z * da) + fb * (b.w + b.z * db);
  return r;
}

// A row's (or a slice's) elements as 16-byte vectors on 16-byte boundaries; what lies outside reads as -inf.
template <typename T>
struct Row {
  static constexpr int kE = 16 / sizeof(T);
  const T* base;       // on a 16-byte boundary, at or before the row
  int first, last;     // elements of the row are [first, last) of base
  __device__ __forceinline__ bool inside(int v) const { return v * kE >= first && v * kE + kE <= last; }
  __device__ __forceinline__ uint4 load(int v) const {
    if (inside(v)) return __ldcs(reinterpret_cast<const uint4*>(base) + v);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(base);
        const int e = v * kE + 2 * i;
        w[i] = (e >= first && e < last ? h[e] : 0xFF80u) | (uint32_t)(e + 1 >= first && e + 1 < last ? h[e + 1] : 0xFF80u) << 16;
      } else {
        const int e = v * kE + i;
        w[i] = e >= first && e < last ? reinterpret_cast<const uint32_t*>(base)[e] : 0xFF800000u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // Elements of a vector as floats.
  static __device__ __forceinline__ void floats(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      else x[i] = __uint_as_float(w[i]);
    }
  }
  static __device__ __forceinline__ float max_of(const uint4& a, const uint4& b, const uint4& c, const uint4& d) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w[16] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w, d.x, d.y, d.z, d.w};
      uint32_t m = w[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
      return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
    } else {
      const uint32_t w[16] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w, d.x, d.y, d.z, d.w};
      float m = __uint_as_float(w[0]);
#pragma unroll
      for (int i = 1; i < 16; ++i) m = max_nan(m, __uint_as_float(w[i]));
      return m;
    }
  }
};

// The order key of a batch's maximum: bfloat16 rows need its upper half alone.
template <typename T>
struct SlotKey {
  typedef uint32_t type;
  static __device__ __forceinline__ uint32_t pack(uint32_t k) { return k; }
  static __device__ __forceinline__ uint32_t unpack(uint32_t k) { return k; }
};
template <>
struct SlotKey<bf16> {
  typedef uint16_t type;
  static __device__ __forceinline__ uint16_t pack(uint32_t k) { return (uint16_t)(k >> 16); }
  // the lower bits of a bfloat16's key: zeros for a positive value, ones for a negative one; 0 stays 0
  static __device__ __forceinline__ uint32_t unpack(uint16_t k) { return (uint32_t)k << 16 | (k - 1u < 0x7FFFu ? 0xFFFFu : 0u); }
};

template <typename T, int kThreads>
struct Shared {
  static constexpr int kWarps = kThreads / 32;
  typename SlotKey<T>::type slot[kSlots][kThreads];   // order keys of the batches' maxima
  __align__(16) unsigned long long cand[kCand];       // order key << 32 | ~index
  unsigned long long list[kMostTop];                  // this CTA's best, in order
  __align__(16) uint32_t best[kThreads];              // order keys of the threads' maxima
  Sums sums[kWarps];
  Sums mine;
  int scan[kWarps + 1];
  uint32_t bound;
  int n_cand, n_list;
};

// Exclusive sum over the CTA's threads.
template <int kWarps>
__device__ __forceinline__ int block_exclusive(int x, int* sh, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh[w];
    all += sh[w];
  }
  *total = all;
  return before + v - x;
}

// The want-th largest of the maxima of kThreads / kEach groups of neighbouring threads (all threads; 1 <= want <= groups).
template <int kEach, int kThreads>
__device__ __forceinline__ uint32_t nth_largest(uint32_t* best, uint32_t* bound, uint32_t mine, int want) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int d = 1; d < kEach; d <<= 1) mine = max(mine, __shfl_xor_sync(~0u, mine, d));
  if (tid % kEach == 0) best[tid / kEach] = mine;
  __syncthreads();
  if (tid < kThreads / kEach) {
    mine = best[tid];
    int above = 0;
    const uint4* all = reinterpret_cast<const uint4*>(best);
#pragma unroll 4
    for (int i = 0; i < kThreads / kEach / 4; ++i) {
      const uint4 k = all[i];
      // of equal keys the lower place's counts as larger: ranks are distinct
      above += (k.x > mine || (k.x == mine && 4 * i < tid)) + (k.y > mine || (k.y == mine && 4 * i + 1 < tid)) +
               (k.z > mine || (k.z == mine && 4 * i + 2 < tid)) + (k.w > mine || (k.w == mine && 4 * i + 3 < tid));
    }
    if (above == want - 1) *bound = mine;
  }
  __syncthreads();
  return *bound;
}

// The top_n largest elements of the slice into s.list (all threads); n_list of them.
template <typename T, int kThreads>
__device__ __noinline__ void select_top(Shared<T, kThreads>& s, const Row<T>& row, int v0, int v1, int rounds_per_slot,
                                        int slots, int top_n, uint32_t mine) {
  constexpr int kE = Row<T>::kE, kWarps = kThreads / 32;
  const int tid = threadIdx.x;
  const int size = min(v1 * kE, row.last) - max(v0 * kE, row.first);   // elements of the slice
  const int want = min(top_n, max(size, 0));
  if (want == 0) return;
  // mine: the order key of the thread's maximum; 0, below that of -inf, without an element: with fewer threads at work than
  // elements wanted all elements count
  // groups of 4 threads give nearly as good a bound for few elements and cost a sixteenth of the comparisons
  const uint32_t t = want <= kThreads / 8 ? nth_largest<4, kThreads>(s.best, &s.bound, mine, want)
                                          : nth_largest<1, kThreads>(s.best, &s.bound, mine, want);
  const int per = rounds_per_slot;
  // This thread's elements of a slot that are at least `from`.  The comparisons go without branches and the few hits are
  // read again: this code runs once a row, and a short one costs its instruction fetches (a branch with its body for every
  // element of a batch took 9 us of a row's 40).
  auto each = [&](int slot, uint32_t from, auto&& f) {
    const float least = from == 0 ? -INFINITY : key_value(from);
#pragma unroll 1
    for (int r = slot * per; r < slot * per + per; ++r) {
      uint4 u[4];
      const int v = v0 + r * 4 * kThreads + tid;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = v + j * kThreads < v1 ? row.load(v + j * kThreads) : make_uint4(0, 0, 0, 0);
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x[kE];
        Row<T>::floats(u[j], x);
#pragma unroll
        for (int e = 0; e < kE; ++e) hits |= x[e] >= least ? 1u << (j * kE + e) : 0u;
      }
#pragma unroll 1
      for (; hits; hits &= hits - 1) {
        const int b = __ffs(hits) - 1, w = v + b / kE * kThreads, i = w * kE + b % kE;
        if (w >= v1 || i < row.first || i >= row.last) continue;
        const uint32_t k = order_key(to_f(row.base[i]));
        if (k >= from) f(k, i - row.first);
      }
    }
  };
  auto collect = [&](uint32_t from) {     // all elements of that key or above; how many
    if (tid == 0) s.n_cand = 0;
    __syncthreads();
    uint32_t mask = 0;
    for (int i = 0; mine >= from && i < slots; ++i) mask |= (uint32_t)(SlotKey<T>::unpack(s.slot[i][tid]) >= from) << i;
    for (; mask; mask &= mask - 1)        // the lanes of a warp read their own batches at the same time
      each(__ffs(mask) - 1, from, [&](uint32_t k, int at) {
        const int p = atomicAdd(&s.n_cand, 1);
        if (p < kCand) s.cand[p] = ((unsigned long long)k << 32) | (uint32_t)~at;
      });
    __syncthreads();
    return s.n_cand;
  };
  int n = 0;
#pragma unroll 1
  for (uint32_t from = t; from <= t + 1; ++from) {   // so many equal to t: those above it, then the equal ones by index
    __syncthreads();
    if ((n = collect(from)) <= kCand) break;
  }
  if (n > kCand) {
    // too many above t in a few batches: one after the other
    unsigned long long below = ~0ull;
    for (int k = 0; k < want; ++k) {
      unsigned long long best = 0;
      for (int i = 0; i < slots; ++i)
        each(i, 0u, [&](uint32_t key, int at) {
          const unsigned long long c = ((unsigned long long)key << 32) | (uint32_t)~at;
          if (c < below && c > best) best = c;
        });
      for (int d = 16; d; d >>= 1) {
        const unsigned long long o = __shfl_xor_sync(~0u, best, d);
        best = o > best ? o : best;
      }
      __syncthreads();
      if ((tid & 31) == 0) s.cand[tid >> 5] = best;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) best = s.cand[w] > best ? s.cand[w] : best;
      below = best;
      if (tid == 0) s.list[k] = best, s.n_list = k + 1;
    }
    __syncthreads();
    return;
  }
  // the candidates' ranks; the best go to the list
  for (int i = tid; i < n; i += kThreads) {
    const unsigned long long c = s.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.cand[j] > c;
    if (rank < want) s.list[rank] = c;
  }
  if (n < want) {   // elements equal to t, by index: rounds in order, in a round the vectors in order
    int found = n;
    for (int i = 0; i < slots && found < want; ++i) {
      const bool holds = SlotKey<T>::unpack(s.slot[i][tid]) >= t;
      if (!__syncthreads_or(holds)) continue;
      for (int r = i * per; r < i * per + per && found < want; ++r)
        for (int j = 0; j < 4 && found < want; ++j) {
          const int v = v0 + (r * 4 + j) * kThreads + tid;
          uint32_t hit = 0;
          if (holds && v < v1) {
            float x[kE];
            Row<T>::floats(row.load(v), x);
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              const int at = v * kE + e;
              if (at >= row.first && at < row.last && order_key(x[e]) == t) hit |= 1u << e;
            }
          }
          int total, p = found + block_exclusive<kWarps>(__popc(hit), s.scan, &total);
          for (; hit && p < want; hit &= hit - 1, ++p)
            s.list[p] = ((unsigned long long)t << 32) | (uint32_t)~(v * kE + __ffs(hit) - 1 - row.first);
          found += total;
        }
    }
  }
  if (tid == 0) s.n_list = want;
  __syncthreads();
}

// Reads the slice: this thread's part of the sums; the batches' maxima where `slot` is given.
template <typename T, int kThreads, bool kCareful>
__device__ __forceinline__ Sums stream(const Row<T>& row, int v0, int v1, int rounds, int per_slot, int slots,
                                       typename SlotKey<T>::type* slot) {
  constexpr int kE = Row<T>::kE;
  constexpr float kLog2e = 1.4426950408889634f;
  const int tid = threadIdx.x;
  float m = -INFINITY, ref = -INFINITY;     // ref: K, or (careful) m itself
  uint64_t z2 = pack2(0.f, 0.f), w2 = z2;   // even and odd elements
  const uint64_t c2 = pack2(kLog2e, kLog2e);
  uint64_t nr = 0;
  const uint4 none = sizeof(T) == 2 ? make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u)
                                    : make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
  float floor = 0.f;                        // far enough below m: a term of 0, and no infinity in a product with 0
  uint32_t floor2 = 0;
  int round = 0;
  const int fast_to = (v1 - v0) / (4 * kThreads) - !row.inside(v1 - 1);   // rounds of whole vectors, but the first
  const uint4* p = reinterpret_cast<const uint4*>(row.base) + v0 + tid;
  uint4 next[4] = {none, none, none, none};
  bool ahead = false;
  for (int i = 0; i < slots; ++i) {
    float slot_max = -INFINITY;
    bool any = false;
    for (int k = 0; k < per_slot && round < rounds; ++k, ++round) {
      uint4 u[4];
      const int v = v0 + round * 4 * kThreads + tid;
      if (ahead) {
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = next[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = v + j * kThreads < v1 ? row.load(v + j * kThreads) : none;
      }
      any |= v < v1;
      ahead = round + 1 < fast_to;        // the next round's vectors are under way while this one's are summed
      if (ahead) {
#pragma unroll
        for (int j = 0; j < 4; ++j) next[j] = __ldg(p + (j + 4) * kThreads);
      }
      p += 4 * kThreads;
      const float bm = Row<T>::max_of(u[0], u[1], u[2], u[3]);
      slot_max = max_nan(slot_max, bm);
      if (!(bm <= m)) {                     // a new maximum (or NaN)
        const float old = ref;
        const bool had = m != -INFINITY;
        m = max_nan(m, bm);
        ref = kCareful ? m : m * kLog2e;
        floor = m - 16384.f;
        floor2 = pack_bf16x2(floor, floor);
        nr = pack2(-ref, -ref);
        if (had) {
          const float d = fmaxf(old - ref, -1e30f), f = exp2_f(kCareful ? d * kLog2e : d);
          w2 = mul2(pack2(f, f), fma2(z2, pack2(d, d), w2));
          z2 = mul2(pack2(f, f), z2);
        }
      }
      if (!kCareful && m == -INFINITY) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float e[kE];
        if constexpr (kCareful) {
          Row<T>::floats(u[j], e);
        } else if constexpr (sizeof(T) == 2) {
          uint4 x;
          asm("max.bf16x2 %0, %1, %2;" : "=r"(x.x) : "r"(u[j].x), "r"(floor2));
          asm("max.bf16x2 %0, %1, %2;" : "=r"(x.y) : "r"(u[j].y), "r"(floor2));
          asm("max.bf16x2 %0, %1, %2;" : "=r"(x.z) : "r"(u[j].z), "r"(floor2));
          asm("max.bf16x2 %0, %1, %2;" : "=r"(x.w) : "r"(u[j].w), "r"(floor2));
          Row<T>::floats(x, e);
        } else {
          Row<T>::floats(u[j], e);
#pragma unroll
          for (int p = 0; p < kE; ++p) e[p] = fmaxf(e[p], floor);
        }
#pragma unroll
        for (int p = 0; p < kE; p += 2) {
          float y0, y1;
          uint64_t d;
          if constexpr (kCareful) {
            unpack2(add2(pack2(e[p], e[p + 1]), nr), y0, y1);
            d = pack2(fmaxf(y0, -1e30f), fmaxf(y1, -1e30f));
            unpack2(mul2(d, c2), y0, y1);
          } else {
            d = fma2(pack2(e[p], e[p + 1]), c2, nr);
            unpack2(d, y0, y1);
          }
          const uint64_t y = pack2(exp2_f(y0), exp2_f(y1));
          z2 = add2(z2, y);
          w2 = fma2(y, d, w2);
        }
      }
    }
    if (slot) slot[i * kThreads + tid] = SlotKey<T>::pack(any ? order_key(slot_max) : 0u);
  }
  Sums t;
  float a0, a1;
  t.m = m;
  // K is m times the float32 constant, not times log2(e): its inverse takes it back.  ln 2 would leave 1.3e-8 of the row's level
  // in every log probability (1.1e-4 at 8000).
  t.ref = kCareful ? (double)ref : (double)ref * (1.0 / (double)kLog2e);
  unpack2(z2, a0, a1);
  t.z = a0 + a1;
  unpack2(w2, a0, a1);
  t.w = kCareful ? a0 + a1 : (a0 + a1) * 0.6931471805599453f;
  return t;
}
template <typename T, int kThreads>
__device__ __noinline__ Sums stream_careful(const Row<T>& row, int v0, int v1, int rounds, int per_slot, int slots) {
  return stream<T, kThreads, true>(row, v0, v1, rounds, per_slot, slots, nullptr);
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) log_probs_kernel(const jx_log_probs_args a, int rounds_per_slot) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared<T, kThreads>& s = *reinterpret_cast<Shared<T, kThreads>*>(smem);
  constexpr int kE = Row<T>::kE, kWarps = kThreads / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const int r = blockIdx.x / C;
  const T* x = static_cast<const T*>(a.logits) + (long long)r * a.ld;
  Row<T> row;
  row.first = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  row.base = x - row.first;
  row.last = row.first + a.V;
  const int nv = (row.last + kE - 1) / kE;
  const int v0 = (int)((long long)nv * rank / C), v1 = (int)((long long)nv * (rank + 1) / C);
  const int rounds = (v1 - v0 + 4 * kThreads - 1) / (4 * kThreads);
  const int slots = (rounds + rounds_per_slot - 1) / rounds_per_slot;

  // the given token's logit on its way while the row is read
  int id = -1;
  float given = 0.f;
  if (rank == 0 && tid == 0) {
    id = a.ids[r];
    if (id >= 0 && id < a.V) given = to_f(x[id]);
  }
  Sums t = stream<T, kThreads, false>(row, v0, v1, rounds, rounds_per_slot, slots, a.top_n ? &s.slot[0][0] : nullptr);
  if (__syncthreads_or(t.m != -INFINITY && !(fabsf(t.m) <= 8192.f)))
    t = stream_careful<T, kThreads>(row, v0, v1, rounds, rounds_per_slot, slots);
  const uint32_t my_key = v0 + tid < v1 ? order_key(t.m) : 0u;
  const bool no_order = __syncthreads_or(t.m != t.m);    // NaN
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    Sums o;
    o.ref = __shfl_xor_sync(~0u, t.ref, d), o.m = __shfl_xor_sync(~0u, t.m, d);
    o.z = __shfl_xor_sync(~0u, t.z, d), o.w = __shfl_xor_sync(~0u, t.w, d);
    // the lower lane's first on both sides: one result for the warp
    t = lane & d ? joined(o, t) : joined(t, o);
  }
  if (lane == 0) s.sums[warp] = t;
  if (tid == 0) s.n_list = 0;
  __syncthreads();
  if (warp == 0) {
    t = s.sums[lane & (kWarps - 1)];
#pragma unroll
    for (int d = kWarps / 2; d; d >>= 1) {
      Sums o;
      o.ref = __shfl_xor_sync(~0u, t.ref, d), o.m = __shfl_xor_sync(~0u, t.m, d);
      o.z = __shfl_xor_sync(~0u, t.z, d), o.w = __shfl_xor_sync(~0u, t.w, d);
      t = lane & d ? joined(o, t) : joined(t, o);
    }
    if (lane == 0) s.mine = t;
  }
  if (a.top_n && !no_order) select_top<T, kThreads>(s, row, v0, v1, rounds_per_slot, slots, a.top_n, my_key);
  if (C > 1) {
    cluster_sync_all();
    if (rank == 0) {
      if (tid == 0) {
        t = s.mine;
        for (int q = 1; q < C; ++q) {
          const uint32_t at = dsmem_map(smem_u32(&s.mine), q);
          Sums o;
          o.ref = __hiloint2double(__float_as_int(dsmem_ld_f32(at + 4)), __float_as_int(dsmem_ld_f32(at)));
          o.m = dsmem_ld_f32(at + 8), o.z = dsmem_ld_f32(at + 12), o.w = dsmem_ld_f32(at + 16);
          t = joined(t, o);
        }
        s.mine = t;
      }
      // every CTA's list behind the others in the candidates
      int n = 0;
      if (a.top_n) {
        for (int q = 0; q < C; ++q) {
          const int have = q == 0 ? s.n_list : __float_as_int(dsmem_ld_f32(dsmem_map(smem_u32(&s.n_list), q)));
          const uint32_t at = dsmem_map(smem_u32(&s.list[0]), q);
          if (tid < have) {
            const uint32_t lo = __float_as_uint(dsmem_ld_f32(at + tid * 8)), hi = __float_as_uint(dsmem_ld_f32(at + tid * 8 + 4));
            s.cand[n + tid] = ((unsigned long long)hi << 32) | lo;
          }
          n += have;
        }
      }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const unsigned long long c = s.cand[i];
        int k = 0;
        for (int j = 0; j < n; ++j) k += s.cand[j] > c;
        if (k < a.top_n) s.list[k] = c;
      }
      __syncthreads();
    }
    cluster_sync_all();      // the others' shared memory is read until here
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  // log p = (x - ref) - log z, the difference in 64 bits: the reference is rounded, and may be large beside it
  t = s.mine;
  const bool fine = t.m == t.m && fabsf(t.m) != INFINITY;
  const float lz = logf(t.z);
  if (tid == 0) {
    a.log_probs[r] = id < 0 ? 0.f : id >= a.V || !fine ? nan_f() : (float)((double)given - t.ref) - lz;
    a.entropy[r] = fine ? lz - t.w / t.z : nan_f();
  }
  if (tid < a.top_n) {
    const bool order = t.m == t.m;
    const unsigned long long c = order ? s.list[tid] : 0;
    a.top_ids[(long long)r * a.top_n + tid] = order ? (int)~(uint32_t)c : -1;
    a.top_log_probs[(long long)r * a.top_n + tid] =
        fine ? (float)((double)key_value((uint32_t)(c >> 32)) - t.ref) - lz : nan_f();
  }
}

template <typename T, int kThreads>
int launch_with(const jx_log_probs_args& a, cudaStream_t s) {
  // CTAs per row: as long as each has a multiprocessor to itself, and its slice two rounds of vectors.  128256 bfloat16
  // logits, top 20, 1 : 2 : 4 : 8 CTAs a row: 7 rows 16.7 : 13.7 : 12.8 : 13.6 us, 37 rows 17.3 : 14.4 : 15.0 : 18.5, 74 rows
  // 17.7 : 14.7 : 18.7 : 29.6, 148 rows 17.5 : 19.4 : 28.8 : 45.6.
  const int e = 16 / (int)sizeof(T);
  int C = 1;
  while (C < 4 && (long long)a.rows * C * 2 <= 148 && a.V / (2 * C) >= 2 * kThreads * 4 * e / 4) C *= 2;
  const long long nv = ((long long)a.V + e - 1) / e + 1;      // a row off its boundary has one vector more
  const long long per_cta = (nv + C - 1) / C;
  const long long rounds = (per_cta + 4 * kThreads - 1) / (4 * kThreads);
  const int per_slot = (int)((rounds + kSlots - 1) / kSlots);
  const int smem = (int)sizeof(Shared<T, kThreads>);
  static bool ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return JX_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(log_probs_kernel<T, kThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return JX_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, log_probs_kernel<T, kThreads>, a, per_slot) == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

template <typename T>
int launch(const jx_log_probs_args& a, cudaStream_t s) {
  // 256 threads a row while all rows are resident at once (4 CTAs a multiprocessor), 128 above: twice the rows in a wave, so
  // fewer of the waits at a row's end are waited for one after the other.  128256 bfloat16 logits, top 20, 256 : 128 threads:
  // 148 rows 17.6 : 22.0 us, 592 rows 40.6 : 44.7, 700 rows 56.7 : 50.4, 1024 rows 71 : 64, 2000 rows 121 : 117; 5000 rows of
  // 32000 139 : 110.
  return a.rows > 4 * 148 ? launch_with<T, 128>(a, s) : launch_with<T, 256>(a, s);
}

}  // namespace

int run_token_log_probs(const jx_log_probs_args& a, cudaStream_t s) {
  return a.dtype == JX_BF16 ? launch<bf16>(a, s) : launch<float>(a, s);
}

}  // namespace jxb
