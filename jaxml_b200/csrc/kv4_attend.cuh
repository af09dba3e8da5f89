// What the attention kernels over the 4-bit KV cache share: arguments, the order of work, operand pieces.
#pragma once

#include <cudaTypedefs.h>
#include <math.h>

#include "kv4.cuh"

namespace jxb {
namespace kv4 {

struct AttendArgs {
  jx_kv4_cache c;
  int layer, S, Hq, G, window, q_vec, items, tiles;   // tiles: query tiles of a row; items = rows * tiles
  float scale_log2, sign;   // |scale| log2(e), at least 1e-30 so that a hidden -inf stays one; its sign, taken into q
  const void* q;
  long long q_row, q_tok, q_head;
  void* out;
  long long* item_first;   // [items] first unit of an item (written by the first CTA)
  long long* total;        // [2] units, warps
  // [runs][2] slots of a tile's rows: O, then (m, l) of each row.  O is [rows][hd], of 128 rows (a thread a row) [hd / 4][128][4]
  float* part;
};

// ---- small pieces -------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t code2(uint32_t w, int k) { return as_u(__hsub2(as_b2(raw2(w, k)), as_b2(0x43084308u))); }
// Whether a pair of scales has one that the format does not (NaN; 2^120 or more): bits to be or'ed and tested against
// 0x80008000.
__device__ __forceinline__ uint32_t bad_scales(uint32_t s2) { return (s2 & 0x7FFF7FFFu) + (0x8000u - kKv4BadScale) * 0x10001u; }
__device__ __forceinline__ void mma_c(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                      float c0, float c1, float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float exp2_f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Where the copy's swizzle puts a byte of a block (16-byte pieces of a 128-byte line exchanged by the line's number).
template <int HD>
__device__ __forceinline__ int swz(int o) {
  return o ^ (((o >> 7) & (HD / 32 - 1)) << 4);
}
__device__ __forceinline__ uint32_t lds16(const unsigned char* p) { return *reinterpret_cast<const uint16_t*>(p); }

// ---- the order of work ------------------------------------------------------------------------------------
// Pages [p0, p0 + n) that query tile `qt` of a row sees.
struct Item {
  int r, qt, cnt, base, n, p0;   // base: position of query 0
};
template <int kRows>
__device__ __forceinline__ Item item_at(const AttendArgs& a, long long item) {
  Item t;
  t.r = (int)(item / a.tiles), t.qt = (int)(item - (long long)t.r * a.tiles);
  // both may be anything in a cache made of given tensors: a difference of two that are not negative does not wrap
  const int cnt = max(a.c.counts[t.r], 0), len = min(max(a.c.lengths[t.r], 0), a.c.row_pages * kPage);
  t.cnt = min(cnt, a.S);
  t.base = len - cnt;
  const int s0 = t.qt * kRows / a.G, s1 = min(min(t.qt * kRows + kRows, a.S * a.G) - 1, t.cnt * a.G - 1) / a.G;
  t.n = 0, t.p0 = 0;
  if (s0 < t.cnt && t.base >= 0) {
    t.p0 = a.window > 0 ? max(0, t.base + s0 - a.window + 1) / kPage : 0;
    t.n = (t.base + s1) / kPage - t.p0 + 1;
  }
  return t;
}

struct Walk {
  Item t;
  long long item;
  int head, page;
  template <int kRows>
  __device__ __forceinline__ void next(const AttendArgs& a) {
    if (++page < t.n) return;
    page = 0;
    if (++head < a.c.num_kv_heads) return;
    head = 0;
    do {
      ++item;
      if (item >= a.items) return;
      t = item_at<kRows>(a, item);
    } while (t.n == 0);
  }
};

// Quotient of two non-negative numbers; most fit 32 bits, where the division is a quarter of the work.
__device__ __forceinline__ long long divide(long long a, long long b) {
  return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
// First unit of run w.
__device__ __forceinline__ long long run_start(long long w, long long units, long long runs) { return divide(w * units, runs); }
// The run that holds unit u.
__device__ __forceinline__ long long run_of(long long u, long long units, long long runs) {
  return divide((u + 1) * runs - 1, units);
}

// ---- loading queries ----------------------------------------------------------------------------------------
// 8 neighbouring channels as they lie in memory.
template <typename T>
struct QPiece {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void load_unaligned(const T* p) {
    __align__(16) T x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(x)[i];
  }
};
// N pieces `step` elements apart, zeros for a row that is not there.  All loads are under way together: one after the other
// they were 16 trips to memory for a row of 128 channels.
template <int N, typename T>
__device__ __forceinline__ void q_load(const T* p, int step, bool live, bool vec, QPiece<T>* q) {
  if (live && vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) q[i].load(p + i * step);
  } else if (live) {
#pragma unroll
    for (int i = 0; i < N; ++i) q[i].load_unaligned(p + i * step);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k) q[i].u[k] = make_uint4(0, 0, 0, 0);
  }
}
// A piece as fragment registers (0,4) (1,5) (2,6) (3,7), a float32 split into 3 parts.
__device__ __forceinline__ void q_words(const QPiece<bf16>& q, float sign, uint4* out) {
  uint32_t x[4] = {q.u[0].x, q.u[0].y, q.u[0].z, q.u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] ^= sign < 0.f ? 0x80008000u : 0u;
  out[0] = make_uint4(__byte_perm(x[0], x[2], 0x5410), __byte_perm(x[0], x[2], 0x7632), __byte_perm(x[1], x[3], 0x5410),
                      __byte_perm(x[1], x[3], 0x7632));
}
__device__ __forceinline__ void q_words(const QPiece<float>& q, float sign, uint4* out) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __uint_as_float(q.u[i].x), x[4 * i + 1] = __uint_as_float(q.u[i].y);
    x[4 * i + 2] = __uint_as_float(q.u[i].z), x[4 * i + 3] = __uint_as_float(q.u[i].w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= sign;
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    out[part] = make_uint4(pack_bf16x2(x[0], x[4]), pack_bf16x2(x[1], x[5]), pack_bf16x2(x[2], x[6]), pack_bf16x2(x[3], x[7]));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] -= rnd<bf16>(x[i]);
  }
}

template <typename T>
__device__ __forceinline__ void store_row8(T* o, const float* x) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(o)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(o)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(o) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                              pack_bf16x2(x[6], x[7]));
  }
}
template <int HD, typename T>
__device__ __forceinline__ T* out_row(const AttendArgs& a, int r, int head, int f) {
  const int s = f / a.G;
  return static_cast<T*>(a.out) + (((long long)r * a.S + s) * a.Hq + head * a.G + (f - s * a.G)) * HD;
}

// A bounded wait on the clock counter (reading the global timer between polls costs more than most waits here last).  The
// thread may be suspended until the phase completes, for some microseconds at a time: a polling warp takes issue slots
// from the others.
constexpr long long kWaitCycles = 4000000000ll;   // about 2 s
__device__ __forceinline__ bool try_wait_long(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_cycles(uint64_t* bar, uint32_t parity) {
  if (try_wait_long(bar, parity)) return true;
  const long long t0 = clock64();
  while (!try_wait_long(bar, parity))
    if (clock64() - t0 > kWaitCycles) return false;
  return true;
}

// Brings the block of a page into shared memory; a page id out of range is reported and its stage marked.
template <int HD>
__device__ __forceinline__ void fetch(const AttendArgs& a, const CUtensorMap* map, int id, int head, unsigned char* to,
                                      uint64_t* bar, int* bad) {
  const bool ok = id >= 0 && id < a.c.num_pages;
  *bad = !ok;
  if (ok) {
    mbar_arrive_expect_tx(bar, kv4_block_bytes(HD));
    tma_load_3d(to, map, 0, 0, (a.layer * a.c.num_pages + id) * a.c.num_kv_heads + head, bar);
  } else {
    set_status(a.c.status, JX_ERR_RANGE);
    mbar_arrive(bar);
  }
}

}  // namespace kv4
}  // namespace jxb
