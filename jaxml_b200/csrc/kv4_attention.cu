// Attention over the pages of the 4-bit KV cache (format in kv4.cuh).
//
// One pass over the keys with a running maximum m and sum l: for a tile of query rows (a query position and a query
// head of one KV head) and a slice of keys,
//   S = K Q^T (keys x rows), P = 2^(S c - m'), O = O 2^(m - m') + V^T P (channels x rows), l = l 2^(m - m') + sum P.
// Both products run on mma.m16n8k16 with the cache as the A operand, so a tile of 8 query rows (the usual decode step:
// the heads that share a KV head) fills the N side and nothing is padded to 16.  The codes go from shared memory
// straight into A fragments: a thread's 32-bit word is 8 neighbouring channels of one key; (w >> 4k) & 0x000F000F is
// the pair (channel k, channel k + 4), a fragment register of K once Q's fragments take the same order, and the same
// bits of two keys' words merged by a byte permute are the pair (key, key + 1) that V^T needs.  0x4300 | u is the
// bfloat16 128 + u.  P changes from the accumulator's layout to the B operand's with movmatrix, without shared memory.
//
// What bounds a decode step is instructions, not bytes: a page of 64 keys is 9 KB and the multiprocessor has some 400
// cycles for it at the card's bandwidth.  So with one tile of 8 rows:
//   K   the k side of an MMA pair is one group of 32 channels, fed with 128 + u; the accumulator starts at
//       -136 sum q of the group and its result times the key's scale is added up in float32 (finite while |q| < 2^115:
//       136 * 32 < 2^13);
//   V   one fused multiply-add a pair gives code times scale exactly (scaled2).
// With more rows K is made exact the same way; float32 results need its codes exact before the product.
//
// Measured (B200, replayed from a graph): 32 rows of 8192 to 16384 tokens, 32 query heads on 8 of 128 features, bf16, 445 MB
// of pages: 125 us, 3.6 TB/s; the copies alone take 87 us, the arithmetic alone some 120: 1430 warp instructions a page, of
// which 800 turn codes into operands.  16 rows of 430 to 768 tokens 11 us, one row of 129 tokens 6.3 us.
//
// A page's block is one tensor-map box of 144 rows of hd / 2 bytes, swizzled by the copy so that ldmatrix gives every
// thread its words of the key it owns without bank conflicts.
#include <algorithm>
#include "kv4_attend.cuh"

namespace jxb {
int run_kv4_attend_tc(const void* args, const void* map, int sms, cudaStream_t s);   // kv4_attention_tc.cu
using namespace kv4;
namespace {

template <int HD, int NT, typename T>
struct Cfg {
  static constexpr int kBlock = kPage * HD + kPage * (HD / 32) * 4;
  static constexpr int kRowBytes = HD / 2;                // a key's codes
  static constexpr int kGroups = HD / 32;
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr bool kRaw = NT == 1 && !kF32;          // codes enter the MMAs with their offset
  static constexpr int kQParts = kF32 ? 3 : 1;            // a float32 as three bfloat16: 24 significant bits
  static constexpr int kPParts = kF32 ? 3 : 1;
  static constexpr int kRows = 8 * NT;
  static constexpr int kVWords = HD / 64;                 // V words of a key and thread
  static constexpr int kMT = HD / 16;
  static constexpr bool kQReg = NT * kQParts * HD / 8 <= 32;
  static constexpr int kQBytes = kQReg ? 0 : NT * kQParts * HD * 16;   // a warp's fragments in shared memory
  static constexpr int kSlot = kRows * (HD + 2);          // floats of a partial result
};

// ---- one tile of query rows over slices of a page -----------------------------------------------------------
template <int HD, int NT, typename T>
struct Tile {
  using C = Cfg<HD, NT, T>;
  float acc[C::kMT][NT][4], m[NT][2], l[NT][2];
  float init[C::kRaw ? C::kGroups : 1][2];        // -136 sum q of a group, columns 2t and 2t + 1 (kRaw)
  int last[NT][2];                                // last visible key of the thread's columns (-1: none)
  uint4 q[C::kQReg ? NT : 1][C::kQReg ? C::kQParts : 1][C::kQReg ? C::kGroups : 1];
  uint4* qs;                                      // the fragments in shared memory otherwise
  int all_hi, all_lo;                             // pages within (all_lo, all_hi] are seen by every row of the tile
  int k_code, v_code[2];                          // the thread's places in a block's codes (swizzled)
  int k_scale, v_scale;                           // and among the scales of 8 keys (not yet)

  __device__ __forceinline__ void begin(const AttendArgs& a, const Item& t, int head, int lane, bool store = true) {
    const int g = lane >> 2, tq = lane & 3, f0 = t.qt * C::kRows, F = a.S * a.G;
    all_hi = f0 + C::kRows <= t.cnt * a.G ? t.base + f0 / a.G : -1;
    all_lo = a.window > 0 ? t.base + (f0 + C::kRows - 1) / a.G - a.window : -1;
    // 8 rows of codes are whole periods of the swizzle: what is added to these places below does not change it
    k_code = HD == 64 ? swz<HD>((((lane >> 4) << 3) + (lane & 7)) * C::kRowBytes + ((lane >> 3) & 1) * 16)
                      : swz<HD>((lane & 7) * C::kRowBytes + (lane >> 3) * 16);
    v_code[0] = swz<HD>(2 * tq * C::kRowBytes + g * (C::kVWords * 4)) + kPage * C::kRowBytes;
    v_code[1] = swz<HD>((2 * tq + 1) * C::kRowBytes + g * (C::kVWords * 4)) + kPage * C::kRowBytes;
    k_scale = g * (HD / 16);
    v_scale = 2 * tq * (HD / 16) + (HD == 64 ? g >> 2 : HD == 128 ? g >> 1 : g) * 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int f = f0 + nt * 8 + 2 * tq + e, s = f / a.G;
        last[nt][e] = f < F && s < t.cnt ? t.base + s : -1;
        m[nt][e] = -INFINITY, l[nt][e] = 0.f;
      }
      const int f = f0 + nt * 8 + g, s = f / a.G;
      const bool live = f < F && s < t.cnt;
      const T* src = static_cast<const T*>(a.q) + t.r * a.q_row + s * a.q_tok + (head * a.G + (f - s * a.G)) * a.q_head;
      constexpr int kTogether = C::kGroups < 4 ? C::kGroups : 4;
      QPiece<T> piece[kTogether];
#pragma unroll
      for (int i = 0; i < C::kGroups; ++i) {
        uint4 x[C::kQParts];
        if (i % kTogether == 0) q_load<kTogether>(src + i * 32 + tq * 8, 32, live, a.q_vec, piece);
        q_words(piece[i % kTogether], a.sign, x);
#pragma unroll
        for (int p = 0; p < C::kQParts; ++p) {
          if constexpr (C::kQReg) q[nt][p][i] = x[p];
          else if (store) qs[((nt * C::kQParts + p) * C::kGroups + i) * 32 + lane] = x[p];
        }
        if constexpr (C::kRaw) {
          float v[8], sum = 0.f;
          unpack8(x[0], v);
#pragma unroll
          for (int k = 0; k < 8; ++k) sum += v[k];
          sum += __shfl_xor_sync(~0u, sum, 1);
          sum += __shfl_xor_sync(~0u, sum, 2);
          init[i][0] = -136.f * __shfl_sync(~0u, sum, tq * 8);
          init[i][1] = -136.f * __shfl_sync(~0u, sum, tq * 8 + 4);
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < C::kMT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][nt][e] = 0.f;
  }

  __device__ __forceinline__ uint4 query(int nt, int p, int grp, int lane) const {
    if constexpr (C::kQReg) return q[nt][p][grp];
    else return qs[((nt * C::kQParts + p) * C::kGroups + grp) * 32 + lane];
  }

  // Place in a scale area (which begins on a whole swizzle period) of byte `o` of the scales of the 8 keys from `key` on.
  static __device__ __forceinline__ int scale_at(int key, int o) {
    const int first = key * (HD / 16);
    return (first & ~127) + (((first & 127) + o) ^ (((first >> 7) & (HD / 32 - 1)) << 4));
  }

  // Keys [kb, kb + KT) of the page in `blk` (shared memory, swizzled), whose first key is key0.  all: every row sees them.
  template <int KT>
  __device__ __forceinline__ void keys(const AttendArgs& a, const unsigned char* blk, int kb, int key0, bool all, int lane) {
    constexpr int kTiles = KT / 16;
    const int g = lane >> 2;
    float sc[kTiles][NT][4];
    const uint32_t base = smem_u32(blk);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      // words of keys g and g + 8: group w's is 4 bytes at 16 w + 4 t of the key's codes
      uint32_t kw[2][C::kGroups];
      const int k16 = kb + i * 16;
      if constexpr (HD == 64) {
        ldsm_x4(base + k_code + k16 * C::kRowBytes, kw[0][0], kw[0][1], kw[1][0], kw[1][1]);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int w = 0; w < C::kGroups; w += 4)   // groups 4..7: the fourth bit of the swizzled piece
            ldsm_x4(base + ((k_code + (k16 + h * 8) * C::kRowBytes) ^ (w * 16)), kw[h][w], kw[h][w + 1], kw[h][w + 2],
                    kw[h][w + 3]);
      }
      uint32_t ks[2][C::kGroups / 2];   // scales of the two keys, two groups a register
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // keys 16 i + 8 h + g: the line, and with it the swizzle, is known but for g's share of it
        const unsigned char* p = blk + kPage * HD + scale_at(k16 + h * 8, k_scale);
        if constexpr (HD == 64) {
          ks[h][0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (HD == 128) {
          const uint2 x = *reinterpret_cast<const uint2*>(p);
          ks[h][0] = x.x, ks[h][1] = x.y;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(p);
          ks[h][0] = x.x, ks[h][1] = x.y, ks[h][2] = x.z, ks[h][3] = x.w;
        }
      }
#pragma unroll
      for (int w = 0; w < C::kGroups; ++w) {
        if constexpr (NT == 1) {
          float x[4];
          uint32_t r[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) r[h][k] = C::kRaw ? raw2(kw[h][w], k) : code2(kw[h][w], k);
#pragma unroll
          for (int p = C::kQParts - 1; p >= 0; --p) {   // the small parts first
            const uint4 b = query(0, p, w, lane);
            if (p == C::kQParts - 1) {
              const float c0 = C::kRaw ? init[w][0] : 0.f, c1 = C::kRaw ? init[w][1] : 0.f;
              mma_c(x, r[0][0], r[1][0], r[0][1], r[1][1], b.x, b.y, c0, c1, c0, c1);
            } else {
              mma_bf16(x, r[0][0], r[1][0], r[0][1], r[1][1], b.x, b.y);
            }
            mma_bf16(x, r[0][2], r[1][2], r[0][3], r[1][3], b.z, b.w);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float s = __uint_as_float(w & 1 ? ks[h][w >> 1] & 0xFFFF0000u : ks[h][w >> 1] << 16);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (w == 0) sc[i][0][2 * h + e] = s * x[2 * h + e];
              else sc[i][0][2 * h + e] = fmaf(s, x[2 * h + e], sc[i][0][2 * h + e]);
            }
          }
        } else {
          uint32_t r[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t s2 = __byte_perm(ks[h][w >> 1], 0, w & 1 ? 0x3232 : 0x1010), c2 = minus136(s2);
#pragma unroll
            for (int k = 0; k < 4; ++k) r[h][k] = scaled2(kw[h][w], k, s2, c2);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float own[4], (&x)[4] = C::kF32 ? own : sc[i][nt];     // float32: a group's products by themselves (Tile)
#pragma unroll
            for (int p = C::kQParts - 1; p >= 0; --p) {
              const uint4 b = query(nt, p, w, lane);
              if ((C::kF32 || w == 0) && p == C::kQParts - 1) mma_c(x, r[0][0], r[1][0], r[0][1], r[1][1], b.x, b.y, 0.f, 0.f, 0.f, 0.f);
              else mma_bf16(x, r[0][0], r[1][0], r[0][1], r[1][1], b.x, b.y);
              mma_bf16(x, r[0][2], r[1][2], r[0][3], r[1][3], b.z, b.w);
            }
            if constexpr (C::kF32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[i][nt][e] = w == 0 ? own[e] : sc[i][nt][e] + own[e];
            }
          }
        }
      }
    }
    // softmax over the keys: registers 0, 1 are key g, 2, 3 key g + 8, of columns 2t and 2t + 1
    uint32_t pf[kTiles][NT][C::kPParts][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = sc[i][nt][2 * h + e];
            if (!all) {
              const int key = key0 + kb + i * 16 + h * 8 + g;
              if (key > last[nt][e] || (a.window > 0 && key <= last[nt][e] - a.window)) x = -INFINITY;
            }
            sc[i][nt][2 * h + e] = x;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 16));
        mx = fmaxf(mx, m[nt][e]);
        const float use = mx == -INFINITY ? 0.f : -mx * a.scale_log2;      // nothing visible yet: every term is 2^-inf
        f[e] = exp2_f(__fmul_rn(m[nt][e], a.scale_log2) + use);    // the reference that the older terms were rounded to
        m[nt][e] = mx;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = exp2_f(fmaf(sc[i][nt][2 * h + e], a.scale_log2, use));
            sc[i][nt][2 * h + e] = x;
            sum += x;
          }
        l[nt][e] = fmaf(l[nt][e], f[e], sum);
      }
      if (__any_sync(~0u, f[0] != 1.f || f[1] != 1.f)) {      // seldom, once a row's maximum has settled
#pragma unroll
        for (int i = 0; i < C::kMT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][nt][e] *= f[e & 1];
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x0 = sc[i][nt][2 * h], x1 = sc[i][nt][2 * h + 1];
#pragma unroll
          for (int p = 0; p < C::kPParts; ++p) {
            // probabilities rounded to bfloat16 (half a step: 2^-9 of their binade's top) for bfloat16 results, split in
            // three for float32 ones
            pf[i][nt][p][h] = transpose8x8(pack_bf16x2(x0, x1));
            if (p + 1 < C::kPParts) x0 -= rnd<bf16>(x0), x1 -= rnd<bf16>(x1);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int k16 = kb + i * 16;
      uint32_t vw[4][C::kVWords], s2[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // keys 2t, 2t + 1, 2t + 8, 2t + 9
        const unsigned char* p = blk + v_code[j & 1] + (k16 + (j >> 1) * 8) * C::kRowBytes;
        if constexpr (C::kVWords == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(p);
          vw[j][0] = x.x, vw[j][1] = x.y, vw[j][2] = x.z, vw[j][3] = x.w;
        } else if constexpr (C::kVWords == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(p);
          vw[j][0] = x.x, vw[j][1] = x.y;
        } else {
          vw[j][0] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // the thread's channels are of one group
        const unsigned char* p = blk + kPage * HD + kPage * (HD / 16);
        s2[h] = lds16(p + scale_at(k16 + h * 8, v_scale)) | (lds16(p + scale_at(k16 + h * 8, v_scale + HD / 16)) << 16);
      }
      const uint32_t c2[2] = {minus136(s2[0]), minus136(s2[1])};
#pragma unroll
      for (int wd = 0; wd < C::kVWords; ++wd) {
        const uint32_t lo0 = __byte_perm(vw[0][wd], vw[1][wd], 0x5410), hi0 = __byte_perm(vw[0][wd], vw[1][wd], 0x7632);
        const uint32_t lo1 = __byte_perm(vw[2][wd], vw[3][wd], 0x5410), hi1 = __byte_perm(vw[2][wd], vw[3][wd], 0x7632);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = scaled2(lo0, k, s2[0], c2[0]), a1 = scaled2(hi0, k, s2[0], c2[0]);
          const uint32_t a2 = scaled2(lo1, k, s2[1], c2[1]), a3 = scaled2(hi1, k, s2[1], c2[1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if constexpr (C::kF32) {
              float x[4];
              mma_c(x, a0, a1, a2, a3, pf[i][nt][C::kPParts - 1][0], pf[i][nt][C::kPParts - 1][1], 0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int p = C::kPParts - 2; p >= 0; --p) mma_bf16(x, a0, a1, a2, a3, pf[i][nt][p][0], pf[i][nt][p][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[wd * 4 + k][nt][e] += x[e];
            } else {
              mma_bf16(acc[wd * 4 + k][nt], a0, a1, a2, a3, pf[i][nt][0][0], pf[i][nt][0][1]);
            }
          }
        }
      }
    }
  }

  // Where a value scale of keys [kb, kb + KT) is none of the format (NaN; 2^120 or more), the rows that see its key get NaN in its channels, and the scale
  // in shared memory becomes 0: a row that does not see the key has P = 0 there, and 0 * NaN would reach it.  Runs before
  // keys().
  template <int KT>
  __device__ __forceinline__ void nan_values(const AttendArgs& a, unsigned char* blk, int kb, int key0, int lane) {
    constexpr int kBytes = KT * (HD / 16), kEach = kBytes >= 512 ? 16 : kBytes >= 256 ? 8 : 4;
    const int at = kPage * HD + kPage * (HD / 16) + kb * (HD / 16), g = lane >> 2;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kBytes; i += kEach * 32) {
      const int o = i + lane * kEach;
      if (o < kBytes) {
        const uint32_t* x = reinterpret_cast<const uint32_t*>(blk + swz<HD>(at + o));
        uint32_t w[4] = {0, 0, 0, 0};
        if constexpr (kEach == 16) {
          const uint4 v = *reinterpret_cast<const uint4*>(x);
          w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (kEach == 8) {
          const uint2 v = *reinterpret_cast<const uint2*>(x);
          w[0] = v.x, w[1] = v.y;
        } else {
          w[0] = *x;
        }
#pragma unroll
        for (int j = 0; j < kEach / 4; ++j) top |= bad_scales(w[j]);
      }
    }
    if (!__any_sync(~0u, top & 0x80008000u)) return;
    const int vg = HD == 64 ? g >> 2 : HD == 128 ? g >> 1 : g;
    for (int key = 0; key < KT; ++key) {
      if ((lds16(blk + swz<HD>(at + key * (HD / 16) + vg * 2)) & 0x7FFFu) < kKv4BadScale) continue;
      const int pos = key0 + kb + key;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (pos <= last[nt][e] && (a.window <= 0 || pos > last[nt][e] - a.window)) {
#pragma unroll
            for (int i = 0; i < C::kMT; ++i) acc[i][nt][e] = acc[i][nt][2 + e] = __uint_as_float(0x7FC00000u);
          }
    }
    __syncwarp();
    for (int i = lane; i < kBytes / 2; i += 32) {
      uint16_t* s = reinterpret_cast<uint16_t*>(blk + swz<HD>(at + i * 2));
      if ((*s & 0x7FFFu) >= kKv4BadScale) *s = 0;
    }
    fence_proxy_async();   // the next copy writes here
    __syncwarp();
  }

  __device__ __forceinline__ bool sees_all(int key0) const { return key0 + kPage - 1 <= all_hi && key0 > all_lo; }

  // The column's sum over the warp; the 8 kVWords channels of the thread and column.
  __device__ __forceinline__ float sum(int nt, int e) const {
    float x = l[nt][e];
    x += __shfl_xor_sync(~0u, x, 4);
    x += __shfl_xor_sync(~0u, x, 8);
    return x + __shfl_xor_sync(~0u, x, 16);
  }
  __device__ __forceinline__ float value(int wd, int k, int nt, int e) const {   // channel k of word wd
    return acc[wd * 4 + (k & 3)][nt][(k >> 2) * 2 + e];
  }
};

// ---- equal runs of pages for every warp ------------------------------------------------------------------------
// All (row, query tile, KV head, page) units in one sequence, cut into equal runs, one for each warp of the grid whatever
// the rows' lengths are.  A warp streams its run's pages through its own ring.  A (row, tile, head) that one warp holds
// whole is written at once; the others leave (m, l, O) for kv4_join_kernel, which joins them in order.
template <int HD, int NT, typename T>
struct Runs {
  using C = Cfg<HD, NT, T>;
  static constexpr int kKeys = NT == 1 ? 64 : 32;          // keys between two updates of the maximum
  static constexpr int kBudget = 223 * 1024;
  static constexpr int kMost = NT == 1 && !C::kF32 && HD <= 128 ? 12 : 8;   // by the registers of a thread
  static constexpr int kFit = kBudget / (2 * C::kBlock + C::kQBytes + 64);  // warps with two pages each
  static constexpr int kWarps = kFit < kMost ? kFit : kMost;
  static constexpr int kDeep = (kBudget / kWarps - C::kQBytes - 64) / C::kBlock;
  static constexpr int kStages = kDeep < 4 ? kDeep : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kSmem = kWarps * (kStages * C::kBlock + C::kQBytes + kStages * 16) + (kThreads + 40) * 8 + 1024;
  static_assert(kSmem <= 227 * 1024 && C::kBlock % (HD * 4) == 0, "shared memory, swizzle alignment");
};

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(Runs<HD, NT, T>::kThreads, 1)
    kv4_attend_runs_kernel(const AttendArgs a, const __grid_constant__ CUtensorMap map) {
  using C = Cfg<HD, NT, T>;
  using R = Runs<HD, NT, T>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* qs = ring + R::kWarps * R::kStages * C::kBlock;
  uint64_t* bars = reinterpret_cast<uint64_t*>(qs + R::kWarps * C::kQBytes);
  int* bad = reinterpret_cast<int*>(bars + R::kWarps * R::kStages);
  long long* first = reinterpret_cast<long long*>(bad + 2 * R::kWarps * R::kStages);   // [kThreads + 1]
  long long* sums = first + R::kThreads + 1;                                           // [32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const jx_kv4_cache& c = a.c;
  if (tid == 0) prefetch_tmap(&map);

  // units before each thread's share of the items, and all of them
  const int each = (a.items + R::kThreads - 1) / R::kThreads;
  const int i0 = min(a.items, tid * each), i1 = min(a.items, i0 + each);
  long long mine = 0;
  for (int i = i0; i < i1; ++i) mine += (long long)item_at<C::kRows>(a, i).n * c.num_kv_heads;
  long long v = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) sums[warp] = v;
  if (tid < R::kWarps * R::kStages) mbar_init(&bars[tid], 1);
  fence_barrier_init();
  __syncthreads();
  long long before = 0, units = 0;
#pragma unroll
  for (int w = 0; w < R::kWarps; ++w) {
    if (w < warp) before += sums[w];
    units += sums[w];
  }
  first[tid] = before + v - mine;
  const long long warps = min((long long)gridDim.x * R::kWarps, max(units, 1ll));
  if (blockIdx.x == 0) {
    long long u = before + v - mine;
    for (int i = i0; i < i1; ++i) {
      a.item_first[i] = u;
      if (c.counts[i / a.tiles] > a.S) set_status(c.status, JX_ERR_RANGE);
      u += (long long)item_at<C::kRows>(a, i).n * c.num_kv_heads;
    }
    if (tid == 0) a.total[0] = units, a.total[1] = warps;
  }
  __syncthreads();

  // neighbouring runs on different multiprocessors: few units still spread over all of them
  const long long w = (long long)warp * gridDim.x + blockIdx.x;
  if (w >= warps || units == 0) return;
  const long long u0 = run_start(w, units, warps), u1 = run_start(w + 1, units, warps);
  Walk rd;
  long long seg_first;   // first unit of the (item, head) at hand
  {
    int lo = 0, hi = R::kThreads - 1;   // last share that begins at or before u0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= u0) lo = mid;
      else hi = mid - 1;
    }
    long long u = first[lo];
    rd.item = (long long)lo * each;
    while (true) {
      rd.t = item_at<C::kRows>(a, rd.item);
      const long long n = (long long)rd.t.n * c.num_kv_heads;
      if (u0 < u + n) break;
      u += n;
      ++rd.item;
    }
    rd.head = (int)((u0 - u) / rd.t.n);
    rd.page = (int)((u0 - u) - (long long)rd.head * rd.t.n);
    seg_first = u0 - rd.page;
  }
  unsigned char* my_ring = ring + warp * R::kStages * C::kBlock;
  uint64_t* my_bar = bars + warp * R::kStages;
  int* my_bad = bad + warp * R::kStages;

  // ahead: the walk of the copies, its next page's id read one step early
  Walk ahead = rd;
  long long ua = u0;
  int next_id = c.table[(long long)ahead.t.r * c.row_pages + ahead.t.p0 + ahead.page];
  auto issue = [&](int stage) {
    if (lane == 0) fetch<HD>(a, &map, next_id, ahead.head, my_ring + stage * C::kBlock, &my_bar[stage], &my_bad[stage]);
    if (++ua < u1) {
      ahead.next<C::kRows>(a);
      next_id = c.table[(long long)ahead.t.r * c.row_pages + ahead.t.p0 + ahead.page];
    }
  };
#pragma unroll
  for (int s = 0; s < R::kStages; ++s)
    if (ua < u1) issue(s);

  Tile<HD, NT, T> tile;
  tile.qs = reinterpret_cast<uint4*>(qs + warp * C::kQBytes);
  bool fresh = true;
  int stage = 0;
  uint32_t phase = 0;
  for (long long u = u0; u < u1; ++u) {
    if (fresh) tile.begin(a, rd.t, rd.head, lane);
    fresh = false;
    const bool arrived = wait_cycles(&my_bar[stage], phase);
    if (!__all_sync(~0u, arrived)) {      // give up: no copy of this warp may be in flight when it ends
      if (lane == 0) set_status(c.status, JX_ERR_TIMEOUT);
      for (int s = 0; s < R::kStages; ++s) wait_cycles(&my_bar[s], s < stage ? phase ^ 1 : phase);
      return;
    }
    unsigned char* blk = my_ring + stage * C::kBlock;
    const int key0 = (rd.t.p0 + rd.page) * kPage;
    if (!my_bad[stage]) {
      const bool all = tile.sees_all(key0);
      tile.template nan_values<kPage>(a, blk, 0, key0, lane);
#pragma unroll 1
      for (int kb = 0; kb < kPage; kb += R::kKeys) tile.template keys<R::kKeys>(a, blk, kb, key0, all, lane);
    }
    __syncwarp();
    if (ua < u1) issue(stage);
    if (++stage == R::kStages) stage = 0, phase ^= 1;

    const bool seg_end = rd.page + 1 == rd.t.n;
    if (seg_end || u + 1 == u1) {
      const bool whole = seg_end && seg_first >= u0;
      const int f0 = rd.t.qt * C::kRows, F = a.S * a.G, g = lane >> 2, t = lane & 3;
      float* slot = a.part + (w * 2 + (seg_first >= u0 ? 1 : 0)) * C::kSlot;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float sum = tile.sum(nt, e);
          const int j = nt * 8 + 2 * t + e, f = f0 + j;
          if (f < F) {
            const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            T* o = out_row<HD, T>(a, rd.t.r, rd.head, f) + g * (C::kVWords * 8);
            float* p = slot + j * HD + g * (C::kVWords * 8);
#pragma unroll
            for (int wd = 0; wd < C::kVWords; ++wd) {
              float x[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) x[k] = tile.value(wd, k, nt, e) * inv;
              if (whole) store_row8<T>(o + wd * 8, x);
              else store_row8<float>(p + wd * 8, x);
            }
            if (!whole && g == 0) slot[C::kRows * HD + 2 * j] = tile.m[nt][e] * a.scale_log2, slot[C::kRows * HD + 2 * j + 1] = sum;
          }
        }
      __syncwarp();
    }
    if (u + 1 < u1) {
      if (seg_end) seg_first = u + 1, fresh = true;
      rd.next<C::kRows>(a);
    }
  }
}

// Joins what several runs hold of one (row, tile, head).  Where a row has a few parts a warp takes kMany query rows, their
// loads under way together; where one row may be spread over the whole grid all warps of a CTA share one.  Rows without a
// visible key are zero.
constexpr int kJoinWarps = 8, kMany = 4;
template <int kW>
__device__ __forceinline__ void load_row(const float* p, float* x) {
  if constexpr (kW == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x, x[1] = v.y;
  } else {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
}
template <int HD, typename T, bool kSpread, bool kTc>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_join_kernel(const AttendArgs a, int rows) {
  constexpr int kR = kSpread ? 1 : kMany, kV = HD / 32;
  pdl_wait();
  __shared__ float sh[kSpread ? kJoinWarps : 1][HD + 2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, Hkv = a.c.num_kv_heads;
  const int item = blockIdx.x / Hkv, head = blockIdx.x - item * Hkv;
  const int j0 = kSpread ? blockIdx.y : (blockIdx.y * kJoinWarps + warp) * kR;
  const long long units = a.total[0], runs = a.total[1];
  const long long first = a.item_first[item], end = item + 1 < a.items ? a.item_first[item + 1] : units;
  const long long n = divide(end - first, Hkv), u0 = first + head * n, u1 = u0 + n;
  const long long w0 = n ? run_of(u0, units, runs) : 0, w1 = n ? run_of(u1 - 1, units, runs) : 0;
  if (n && w0 == w1) return;
  const int r = item / a.tiles, qt = item - r * a.tiles, f0 = qt * rows + j0;
  const int live = min(kR, min(rows - j0, a.S * a.G - f0));
  if (!kSpread && live <= 0) return;
  const long long slot_floats = (long long)rows * (HD + 2);
  float m[kR], l[kR], o[kR][kV];
#pragma unroll
  for (int q = 0; q < kR; ++q) {
    m[q] = -INFINITY, l[q] = 0.f;
#pragma unroll
    for (int i = 0; i < kV; ++i) o[q][i] = 0.f;
  }
  for (long long w = w0 + (kSpread ? warp : 0); n && live > 0 && w <= w1; w += kSpread ? kJoinWarps : 1) {
    // the run that the segment begins in holds it in its second slot
    const float* slot = a.part + (w * 2 + (run_start(w, units, runs) <= u0 ? 1 : 0)) * slot_floats;
    float mw[kR], lw[kR], ow[kR][kV];
#pragma unroll
    for (int q = 0; q < kR; ++q) {
      const int j = j0 + min(q, live - 1);
      mw[q] = slot[rows * HD + 2 * j], lw[q] = slot[rows * HD + 2 * j + 1];
      if constexpr (kTc) {
        constexpr int kW = kV < 4 ? kV : 4;
#pragma unroll
        for (int i = 0; i < kV; i += kW) {
          const int at = lane * kV + i;
          load_row<kW>(slot + (at / 4 * 128 + j) * 4 + at % 4, &ow[q][i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) ow[q][i] = slot[j * HD + lane * kV + i];
      }
    }
#pragma unroll
    for (int q = 0; q < kR; ++q) {
      const float mn = fmaxf(m[q], mw[q]), use = mn == -INFINITY ? 0.f : mn;
      const float fo = exp2_f(m[q] - use), fw = exp2_f(mw[q] - use);
      m[q] = mn;
      l[q] = l[q] * fo + lw[q] * fw;
#pragma unroll
      for (int i = 0; i < kV; ++i) o[q][i] = o[q][i] * fo + ow[q][i] * fw;
    }
  }
  if constexpr (kSpread) {
#pragma unroll
    for (int i = 0; i < kV; ++i) sh[warp][lane * kV + i] = o[0][i];
    if (lane == 0) sh[warp][HD] = m[0], sh[warp][HD + 1] = l[0];
    __syncthreads();
    if (warp || live <= 0) return;
    m[0] = -INFINITY, l[0] = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) m[0] = fmaxf(m[0], sh[w][HD]);
#pragma unroll
    for (int i = 0; i < kV; ++i) o[0][i] = 0.f;
    const float use = m[0] == -INFINITY ? 0.f : m[0];
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      const float fw = exp2_f(sh[w][HD] - use);
      l[0] += sh[w][HD + 1] * fw;
#pragma unroll
      for (int i = 0; i < kV; ++i) o[0][i] += sh[w][lane * kV + i] * fw;
    }
  }
#pragma unroll
  for (int q = 0; q < kR; ++q) {
    if (q >= live) continue;
    T* out = out_row<HD, T>(a, r, head, f0 + q) + lane * kV;
    const float inv = l[q] == 0.f ? 0.f : 1.f / l[q];
#pragma unroll
    for (int i = 0; i < kV; ++i) out[i] = from_f<T>(o[q][i] * inv);
  }
}

// ---- one CTA, or a cluster of them, for every (row, query tile, KV head) ----------------------------------------
// A CTA takes its share of the pages; slices of 16 keys go round its warps and their results meet in shared memory, those
// of a cluster's CTAs in each other's: one launch, and the shortest way from the page table to the result.
template <int HD, int NT, typename T>
struct Group {
  using C = Cfg<HD, NT, T>;
  static constexpr int kWarps = 8, kKeys = 16, kThreads = kWarps * 32;
  static constexpr int kPages = HD == 64 ? 8 : 4;          // pages in shared memory at a time
  static constexpr int kJoin = kWarps * C::kSlot * 4;
  static constexpr int kRing = kPages * C::kBlock > kJoin ? kPages * C::kBlock : kJoin;
  static constexpr int kSmem = kRing + C::kQBytes + kPages * 16 + C::kSlot * 4 + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(Group<HD, NT, T>::kThreads)
    kv4_attend_group_kernel(const AttendArgs a, const __grid_constant__ CUtensorMap map) {
  using C = Cfg<HD, NT, T>;
  using R = Group<HD, NT, T>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* qs = ring + R::kRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(qs + C::kQBytes);
  int* bad = reinterpret_cast<int*>(bars + R::kPages);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const jx_kv4_cache& c = a.c;
  float* mine = reinterpret_cast<float*>(bad + 2 * R::kPages);      // [kSlot] this CTA's (O, m, l)
  const int cs = (int)cluster_nctarank(), rank = (int)cluster_ctarank(), seg = blockIdx.x / cs;
  const int item = seg / c.num_kv_heads, head = seg - item * c.num_kv_heads;
  Item t = item_at<C::kRows>(a, item);
  const int f0 = t.qt * C::kRows, rows = min(C::kRows, a.S * a.G - f0);
  if (tid == 0) {
    prefetch_tmap(&map);
    if (c.counts[t.r] > a.S) set_status(c.status, JX_ERR_RANGE);
  }
  if (t.n == 0) {
    for (int i = tid; rank == 0 && i < rows * HD; i += R::kThreads)
      out_row<HD, T>(a, t.r, head, f0 + i / HD)[i % HD] = from_f<T>(0.f);
    return;
  }
  {                                     // this CTA's pages
    const int p = t.n * rank / cs, q = t.n * (rank + 1) / cs;
    t.p0 += p, t.n = q - p;
  }
  int id = -1;
  if (tid < R::kPages) {
    mbar_init(&bars[tid], 1);
    fence_barrier_init();
    if (tid < t.n) {
      id = c.table[(long long)t.r * c.row_pages + t.p0 + tid];
      fetch<HD>(a, &map, id, head, ring + tid * C::kBlock, &bars[tid], &bad[tid]);
    }
  }
  Tile<HD, NT, T> tile;
  tile.qs = reinterpret_cast<uint4*>(qs);   // one copy for all warps
  tile.begin(a, t, head, lane, warp == 0);
  __syncthreads();
  bool dead = false;
  for (int first = 0, phase = 0; first < t.n; first += R::kPages, phase ^= 1) {
    const int here = min(R::kPages, t.n - first);
    for (int sl = warp; sl < here * (kPage / R::kKeys); sl += R::kWarps) {
      const int page = sl / (kPage / R::kKeys), kb = sl % (kPage / R::kKeys) * R::kKeys;
      if (!dead && !__all_sync(~0u, wait_cycles(&bars[page], phase))) {
        dead = true;
        wait_cycles(&bars[page], phase);   // no copy may be in flight when the CTA ends
        if (lane == 0) set_status(c.status, JX_ERR_TIMEOUT);
      }
      unsigned char* blk = ring + page * C::kBlock;
      const int key0 = (t.p0 + first + page) * kPage;
      if (!dead && !bad[page]) {
        tile.template nan_values<R::kKeys>(a, blk, kb, key0, lane);
        tile.template keys<R::kKeys>(a, blk, kb, key0, tile.sees_all(key0), lane);
      }
    }
    __syncthreads();
    if (tid < R::kPages && first + R::kPages + tid < t.n) {
      id = c.table[(long long)t.r * c.row_pages + t.p0 + first + R::kPages + tid];
      wait_cycles(&bars[tid], phase);   // passed already, unless a warp gave up on it
      fetch<HD>(a, &map, id, head, ring + tid * C::kBlock, &bars[tid], &bad[tid]);
    }
    if (first + R::kPages < t.n) __syncthreads();
  }
  float* slots = reinterpret_cast<float*>(ring);
  {
    float* slot = slots + warp * C::kSlot;
    const int g = lane >> 2, tq = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float sum = tile.sum(nt, e);
        const int j = nt * 8 + 2 * tq + e;
        if (j < rows) {
#pragma unroll
          for (int wd = 0; wd < C::kVWords; ++wd) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = tile.value(wd, k, nt, e);
            store_row8<float>(slot + j * HD + (g * C::kVWords + wd) * 8, x);
          }
          if (g == 0) slot[C::kRows * HD + 2 * j] = tile.m[nt][e] * a.scale_log2, slot[C::kRows * HD + 2 * j + 1] = sum;
        }
      }
  }
  __syncthreads();
  const int busy = min(R::kWarps, t.n * (kPage / R::kKeys));   // warps that had a slice
  for (int i = tid; i < rows * (HD / 8); i += R::kThreads) {
    const int j = i / (HD / 8), d = i % (HD / 8) * 8;
    float mx = -INFINITY, sum = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < busy; ++w) mx = fmaxf(mx, slots[w * C::kSlot + C::kRows * HD + 2 * j]);
    const float use = mx == -INFINITY ? 0.f : mx;
    for (int w = 0; w < busy; ++w) {
      const float* slot = slots + w * C::kSlot;
      const float f = exp2_f(slot[C::kRows * HD + 2 * j] - use);
      sum = fmaf(slot[C::kRows * HD + 2 * j + 1], f, sum);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = fmaf(slot[j * HD + d + k], f, x[k]);
    }
    if (cs == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= inv;
      store_row8<T>(out_row<HD, T>(a, t.r, head, f0 + j) + d, x);
    } else {
      store_row8<float>(mine + j * HD + d, x);
      if (d == 0) mine[C::kRows * HD + 2 * j] = mx, mine[C::kRows * HD + 2 * j + 1] = sum;
    }
  }
  if (cs == 1) return;
  cluster_sync_all();
  for (int i = rank * R::kThreads + tid; i < rows * (HD / 8); i += cs * R::kThreads) {
    const int j = i / (HD / 8), d = i % (HD / 8) * 8;
    const uint32_t ml = smem_u32(mine + C::kRows * HD + 2 * j), at = smem_u32(mine + j * HD + d);
    float mx = -INFINITY, sum = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < cs; ++q) mx = fmaxf(mx, dsmem_ld_f32(dsmem_map(ml, q)));
    const float use = mx == -INFINITY ? 0.f : mx;
    for (int q = 0; q < cs; ++q) {
      const uint32_t mq = dsmem_map(ml, q), oq = dsmem_map(at, q);
      const float f = exp2_f(dsmem_ld_f32(mq) - use);
      sum = fmaf(dsmem_ld_f32(mq + 4), f, sum);
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        float4 o;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w) : "r"(oq + k * 4) : "memory");
        x[k] = fmaf(o.x, f, x[k]), x[k + 1] = fmaf(o.y, f, x[k + 1]);
        x[k + 2] = fmaf(o.z, f, x[k + 2]), x[k + 3] = fmaf(o.w, f, x[k + 3]);
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] *= inv;
    store_row8<T>(out_row<HD, T>(a, t.r, head, f0 + j) + d, x);
  }
  cluster_sync_all();      // the others' shared memory is read until here
}

// ---- host ----------------------------------------------------------------------------------------------------
int sm_count() {
  static int n[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!n[dev] && (cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n[dev] <= 0)) n[dev] = 148;
  return n[dev];
}

struct Layout {
  int nt, tiles;
  int group;             // CTAs per (row, tile, head), 0: equal runs
  bool tc;               // 128 query rows a tile, on tcgen05
  long long items, first_at, part_at, bytes;
};
// Groups or equal runs.  A group has no split to compute and no second launch; its clusters have to be resident at once and
// its CTAs to have few pages each, or equal runs over all of the GPU win.  32 query heads on 8 of 128 features, bf16,
// microseconds group : runs at 256, 768, 2000, 8000, 16000 cached tokens: one row 6.4 : 10.8, 7.2 : 11.4, 8.4 : 12.6,
// 16 : 18.9, 26 : 28; 4 rows 6.8 : 11.2, 7.9 : 11.6, 10.6 : 13.2, 19.7 : 22.7, 32 : 30; 16 rows 6.8 : 11.7, 11.6 : 13.2, and
// 25 : 21 at 2000; 64 rows 15 : 19, 27 : 30, and 62 : 51 at 2000.  With tiles of 16 query rows: one row 7.9 : 11.3, 9.5 : 11.9,
// 10.9 : 13.2; 64 rows 29 : 34, and 52 : 47 at 768.  Clusters that do not fit at once cost twice: 16 rows at 768 tokens take 17
// in clusters of 4, 11.6 in clusters of 2; 4 rows of tiles of 16 at 1020 tokens 26 in clusters of 8, 12.7 in runs.
constexpr int kGroupPages = 4;    // pages a CTA, as long as there is room for larger clusters
constexpr int kGroupMost = 16;    // pages a CTA above which runs win (half of it with tiles of 16 rows)
// Clusters of 1, 2, 4 and 8 CTAs that 148 multiprocessors hold at once with one CTA each (head_dim 256, tiles of 16) and with
// two: a cluster stays within a group of some 16 to 20 multiprocessors.
constexpr int kGroupClusters[2][4] = {{148, 74, 33, 15}, {296, 148, 71, 33}};
// bfloat16 rows of a KV head (S * G) from which they are 128 a tile on tcgen05, instead of tiles of 8 or 16 on mma.sync that
// each read the pages: 12 rows of 2048 tokens, 8 of them in the batch, take 25.2 us against 24.4 (mma.sync), 16 rows 26.3
// either way, 24 rows 27.4 against 45.8, 64 rows 35 against 64; 20 rows of 256 features 40 against 46.
// Short rows stay in groups, tiles of 16, while there are few of them: 16 rows of 20 queries at 256 tokens, 256 CTAs, 15 us
// against 24; one row of 64 queries at 512, 8 clusters, 9.5 against 13.4; 16 rows of 64, 512 CTAs, 20 : 20 at 128 tokens and
// 23 : 28 at 256; 16 rows of 128, 1024 CTAs, 36 : 26.
constexpr int kTcRows = 17, kGroupTiles = 512;
constexpr int kMostCtas = 160, kMostWarps = 12;
Layout layout_of(const jx_kv4_cache& c, int S, int Hq, int window, int dtype) {
  Layout l;
  const int G = Hq / c.num_kv_heads;
  const long long rows = (long long)S * G;
  l.nt = rows <= 8 ? 1 : 2;     // float32 tiles of 32 rows would not fit the registers
  auto tiles = [&](int tile) { l.tiles = (int)((rows + tile - 1) / tile), l.items = (long long)c.num_rows * l.tiles; };
  tiles(8 * l.nt);
  long long pages = c.row_pages;                       // that a row can see
  if (window > 0) pages = std::min(pages, ((long long)window + S - 2) / kPage + 2);
  const long long segs = l.items * c.num_kv_heads;
  const int two = l.nt == 1 && c.head_dim < 256;       // CTAs of a multiprocessor, less one
  int step = 0;
  while (step < 3 && pages > kGroupPages << step && segs <= kGroupClusters[two][step + 1]) ++step;
  l.group = pages <= (l.nt == 1 ? kGroupMost : kGroupMost / 2) << step ? 1 << step : 0;
  const bool many = dtype == JX_BF16 && rows >= kTcRows;
  if (many && segs > kGroupTiles) l.group = 0;
  l.tc = many && !l.group;
  if (l.tc) tiles(128);
  const int tile = l.tc ? 128 : 8 * l.nt;
  l.first_at = 16;
  l.part_at = (l.first_at + l.items * 8 + 15) / 16 * 16;
  const long long slots = l.tc ? 2ll * 2 * kMostCtas : 2ll * kMostCtas * kMostWarps;   // two for every run
  l.bytes = l.group ? 0 : l.part_at + slots * tile * (c.head_dim + 2) * 4;
  return l;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }
  return fn;
}

// The pool as [blocks][144 rows][hd / 2 bytes]; a box is one block, a row as wide as the swizzle.
int make_map(CUtensorMap* map, const jx_kv4_cache& c) {
  auto enc = encoder();
  if (!enc) return JX_ERR_CUDA;
  const cuuint64_t blocks = (cuuint64_t)c.num_layers * c.num_pages * c.num_kv_heads;
  const cuuint64_t dims[3] = {(cuuint64_t)c.head_dim / 2, 144, blocks};
  const cuuint64_t strides[2] = {(cuuint64_t)c.head_dim / 2, (cuuint64_t)kv4_block_bytes(c.head_dim)};
  const cuuint32_t box[3] = {(cuuint32_t)c.head_dim / 2, 144, 1}, one[3] = {1, 1, 1};
  const CUtensorMapSwizzle sw = c.head_dim == 64    ? CU_TENSOR_MAP_SWIZZLE_32B
                                : c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                    : CU_TENSOR_MAP_SWIZZLE_128B;
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c.pages, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? JX_OK : JX_ERR_ARG;
}

// Allows a kernel its shared memory, once per device.
template <typename K>
int allow(K kernel, int bytes, bool (&ready)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return JX_ERR_CUDA;
  if (dev >= 0 && dev < 64 && ready[dev]) return JX_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return JX_ERR_CUDA;
  if (dev >= 0 && dev < 64) ready[dev] = true;
  return JX_OK;
}

// The second kernel, for tiles of `rows` query rows and that many runs.
template <int HD, typename T, bool kTc>
int join(const AttendArgs& a, int rows, int runs, cudaStream_t s) {
  const long long segments = a.items * (long long)a.c.num_kv_heads;
  const int there = a.tiles > 1 || a.S * a.G >= rows ? rows : a.S * a.G;
  // Parts a segment, if they are alike.  A CTA a query row is better from 2 on (64 rows of 2000 tokens, 3.5 parts: 48.0
  // against 50.7 us for the whole call; 128 rows, 1.7 parts: 58.8 against 56.8), in tiles of 128 query rows, where most of
  // its warps have none, from 6 on (4.6 parts: 64.6 against 58.0; 18 parts: 36 against 68).
  const bool few = runs <= (there >= 32 ? 6 : 2) * segments;
  cudaLaunchConfig_t cfg = {};
  const int each = few ? kJoinWarps * kMany : 1;
  cfg.gridDim = dim3((unsigned)segments, (unsigned)((there + each - 1) / each));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return (few ? cudaLaunchKernelEx(&cfg, kv4_join_kernel<HD, T, false, kTc>, a, rows)
              : cudaLaunchKernelEx(&cfg, kv4_join_kernel<HD, T, true, kTc>, a, rows)) == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

template <int HD, int NT, typename T>
int launch(const Layout& l, const AttendArgs& a, const CUtensorMap& map, cudaStream_t s) {
  if (l.group) {
    using R = Group<HD, NT, T>;
    static bool ready[64];
    if (const int rc = allow(kv4_attend_group_kernel<HD, NT, T>, R::kSmem, ready)) return rc;
    if (l.group == 1) {
      kv4_attend_group_kernel<HD, NT, T><<<a.items * a.c.num_kv_heads, R::kThreads, R::kSmem, s>>>(a, map);
      return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.items * a.c.num_kv_heads * l.group));
    cfg.blockDim = dim3(R::kThreads);
    cfg.dynamicSmemBytes = R::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = l.group, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_attend_group_kernel<HD, NT, T>, a, map) == cudaSuccess ? JX_OK : JX_ERR_CUDA;
  }
  using R = Runs<HD, NT, T>;
  static_assert(R::kWarps <= kMostWarps, "workspace");
  static bool ready[64];
  if (const int rc = allow(kv4_attend_runs_kernel<HD, NT, T>, R::kSmem, ready)) return rc;
  const long long most = (long long)a.items * a.c.row_pages * a.c.num_kv_heads;   // units there can be
  int grid = sm_count() < kMostCtas ? sm_count() : kMostCtas;
  if (most < grid) grid = (int)most;
  kv4_attend_runs_kernel<HD, NT, T><<<grid, R::kThreads, R::kSmem, s>>>(a, map);
  if (cudaPeekAtLastError() != cudaSuccess) return JX_ERR_CUDA;
  return join<HD, T, false>(a, Cfg<HD, NT, T>::kRows, grid * R::kWarps, s);
}

template <int HD, typename T>
int launch_nt(const Layout& l, const AttendArgs& a, const CUtensorMap& map, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (l.tc) {
      const int sms = sm_count() < kMostCtas ? sm_count() : kMostCtas;
      if (const int rc = run_kv4_attend_tc(&a, &map, sms, s)) return rc;
      return join<HD, T, true>(a, 128, HD == 256 ? sms : 2 * sms, s);
    }
  if (l.nt == 1) return launch<HD, 1, T>(l, a, map, s);
  return launch<HD, 2, T>(l, a, map, s);
}

template <typename T>
int launch_hd(const Layout& l, const AttendArgs& a, const CUtensorMap& map, cudaStream_t s) {
  if (a.c.head_dim == 64) return launch_nt<64, T>(l, a, map, s);
  if (a.c.head_dim == 128) return launch_nt<128, T>(l, a, map, s);
  return launch_nt<256, T>(l, a, map, s);
}

}  // namespace

// Enough for any window: fewer pages turn runs and tiles of 128 into groups, which need none, and nothing else.
long long kv4_attend_workspace(const jx_kv4_cache& c, int S, int Hq, int dtype) { return layout_of(c, S, Hq, 0, dtype).bytes; }

int run_kv4_attend(const jx_kv4_cache& c, int layer, int S, int Hq, const void* q, const long long* qs, void* out,
                   float scale, int window, void* ws, int dtype, cudaStream_t s) {
  const Layout l = layout_of(c, S, Hq, window, dtype);
  AttendArgs a;
  a.c = c, a.layer = layer, a.S = S, a.Hq = Hq, a.G = Hq / c.num_kv_heads, a.window = window;
  a.items = (int)l.items, a.tiles = l.tiles, a.sign = scale < 0.f ? -1.f : 1.f;
  a.scale_log2 = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f);
  a.q = q, a.q_row = qs[0], a.q_tok = qs[1], a.q_head = qs[2], a.out = out;
  const int unit = dtype == JX_BF16 ? 8 : 4;
  a.q_vec = !((uintptr_t)q & 15) && !(qs[0] % unit) && !(qs[1] % unit) && !(qs[2] % unit);
  unsigned char* b = static_cast<unsigned char*>(ws);
  a.total = reinterpret_cast<long long*>(b);
  a.item_first = reinterpret_cast<long long*>(b + l.first_at);
  a.part = reinterpret_cast<float*>(b + l.part_at);
  CUtensorMap map;
  if (const int rc = make_map(&map, c)) return rc;
  return dtype == JX_BF16 ? launch_hd<bf16>(l, a, map, s) : launch_hd<float>(l, a, map, s);
}

}  // namespace jxb
