// Attention over the pages of the 4-bit KV cache (format in kv4.cuh).
//
// One pass over the keys with a running maximum m and sum l: for a tile of query rows (a query position and a query
// head of one KV head) and a page of 64 keys,
//   S = K Q^T (keys x rows), P = 2^(S c - m'), O = O 2^(m - m') + V^T P (channels x rows), l = l 2^(m - m') + sum P.
// Both products run on mma.m16n8k16 with the cache as the A operand, so a tile of 8 query rows (the usual decode step:
// the heads that share a KV head) fills the N side and nothing is padded to 16.  The codes go from shared memory
// straight into A fragments: a thread's 32-bit word is 8 neighbouring channels of one key; (w >> 4k) & 0x000F000F is the pair
// (channel k, channel k + 4), a fragment register of K once Q's fragments take the same order, and the same bits of
// two keys' words merged by a byte permute are the pair (key, key + 1) that V^T needs.  0x4300 | u is bfloat16 128 + u,
// so u - 8 and its product with the scale are exact.  P changes from the accumulator's layout to the B operand's with
// movmatrix, without shared memory.
//
// Work is split into pages: all (row, query tile, KV head, page) units in one sequence, cut into equal runs, one for
// each warp of the grid whatever the rows' lengths are.  A warp streams its run's pages (one bulk copy each: a page's
// block is contiguous) through its own ring.  A (row, tile, head) that one warp holds whole is written at once; the
// others leave (m, l, O) for a second kernel, which joins them in order.
#include <math.h>

#include "kv4.cuh"

namespace jxb {
namespace {

struct AttendArgs {
  jx_kv4_cache c;
  int layer, S, Hq, G, window, q_vec, items, tiles;   // tiles: query tiles of a row; items = rows * tiles
  float scale_log2;
  const void* q;
  long long q_row, q_tok, q_head;
  void* out;
  long long* item_first;   // [items] first unit of an item (written by the first CTA)
  long long* total;        // [2] units, warps
  float* part;             // [warps][2] slots of 8 * NT rows: O, then m and l
};

template <int HD, int NT, typename T>
struct Cfg {
  static constexpr int kBlock = kPage * HD + kPage * (HD / 32) * 4;
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kQParts = kF32 ? 3 : 1;            // a float32 as three bfloat16: 24 significant bits
  static constexpr int kPParts = kF32 ? 3 : 1;
  static constexpr int kRows = 8 * NT;
  static constexpr int kChunks = HD >= 128 ? HD / 128 : 1;
  static constexpr int kWords = HD >= 128 ? 4 : 2;        // K words of a key, chunk and thread
  static constexpr int kVWords = HD / 64;                 // V words of a key and thread
  static constexpr int kMT = HD / 16;
  static constexpr int kKeys = NT == 1 ? 64 : 32;         // keys between two updates of the maximum
  static constexpr bool kQReg = NT * kQParts * HD / 8 <= 32;
  static constexpr int kQBytes = kQReg ? 0 : NT * kQParts * HD * 16;
  static constexpr int kBudget = 224 * 1024;
  static constexpr int kFit = kBudget / (2 * kBlock + kQBytes + 64);   // warps with two pages each
  static constexpr int kWarps = kFit < 8 ? kFit : 8;
  static constexpr int kDeep = (kBudget / kWarps - kQBytes - 64) / kBlock;
  static constexpr int kStages = kDeep < 4 ? kDeep : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kSlot = kRows * (HD + 2);          // floats
  static constexpr int kSmem = kWarps * (kStages * kBlock + kQBytes + kStages * 16) + (kThreads + 40) * 8;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// ---- small pieces -------------------------------------------------------------------------------------
// bfloat16 pair (n_k, n_k+4) - 8 of a word.
__device__ __forceinline__ __nv_bfloat162 codes(uint32_t w, int k) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000F000F, 0x43004300, 0xEA;" : "=r"(r) : "r"(w >> (4 * k)));
  const uint32_t c = 0x43084308u;   // 136
  return __hsub2(*reinterpret_cast<__nv_bfloat162*>(&r), *reinterpret_cast<const __nv_bfloat162*>(&c));
}
__device__ __forceinline__ uint32_t scaled(uint32_t w, int k, uint32_t s2) {
  const __nv_bfloat162 r = __hmul2(codes(w, k), *reinterpret_cast<__nv_bfloat162*>(&s2));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float exp2_f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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
  t.cnt = min(a.c.counts[t.r], a.S);
  const int len = min(a.c.lengths[t.r], a.c.row_pages * kPage);
  t.base = len - a.c.counts[t.r];
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

// First unit of warp w's run.
__device__ __forceinline__ long long run_start(long long w, long long units, long long warps) { return w * units / warps; }
// Warp whose run holds unit u.
__device__ __forceinline__ long long run_of(long long u, long long units, long long warps) {
  return ((u + 1) * warps - 1) / units;
}

// ---- loading queries ----------------------------------------------------------------------------------------
// 8 neighbouring channels as fragment registers (0,4) (1,5) (2,6) (3,7), a float32 split into `parts`.
__device__ __forceinline__ void q_words(const bf16* p, bool vec, uint4* out) {
  uint32_t x[4];
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
  }
  out[0] = make_uint4(__byte_perm(x[0], x[2], 0x5410), __byte_perm(x[0], x[2], 0x7632), __byte_perm(x[1], x[3], 0x5410),
                      __byte_perm(x[1], x[3], 0x7632));
}
__device__ __forceinline__ void q_words(const float* p, bool vec, uint4* out) {
  float x[8];
  if (vec) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    out[part] = make_uint4(pack_bf16x2(x[0], x[4]), pack_bf16x2(x[1], x[5]), pack_bf16x2(x[2], x[6]), pack_bf16x2(x[3], x[7]));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] -= rnd<bf16>(x[i]);
  }
}

// ---- the kernel ---------------------------------------------------------------------------------------------
template <int HD, int NT, typename T>
__global__ void __launch_bounds__(Cfg<HD, NT, T>::kThreads, 1) kv4_attend_kernel(const AttendArgs a) {
  using C = Cfg<HD, NT, T>;
  constexpr int kTiles = C::kKeys / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* ring = smem;
  unsigned char* qs = ring + C::kWarps * C::kStages * C::kBlock;
  uint64_t* bars = reinterpret_cast<uint64_t*>(qs + C::kWarps * C::kQBytes);
  int* bad = reinterpret_cast<int*>(bars + C::kWarps * C::kStages);
  long long* first = reinterpret_cast<long long*>(bad + 2 * C::kWarps * C::kStages);   // [kThreads + 1]
  long long* sums = first + C::kThreads + 1;                                           // [32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const jx_kv4_cache& c = a.c;

  // units before each thread's share of the items, and all of them
  const int each = (a.items + C::kThreads - 1) / C::kThreads;
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
  if (tid < C::kWarps * C::kStages) mbar_init(&bars[tid], 1);
  if (tid == 0) fence_barrier_init();
  __syncthreads();
  long long before = 0, units = 0;
#pragma unroll
  for (int w = 0; w < C::kWarps; ++w) {
    if (w < warp) before += sums[w];
    units += sums[w];
  }
  first[tid] = before + v - mine;
  if (tid == C::kThreads - 1) first[C::kThreads] = units;
  const long long warps = min((long long)gridDim.x * C::kWarps, max(units, 1ll));
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
    int lo = 0, hi = C::kThreads - 1;   // last share that begins at or before u0
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
  unsigned char* my_ring = ring + warp * C::kStages * C::kBlock;
  uint64_t* my_bar = bars + warp * C::kStages;
  int* my_bad = bad + warp * C::kStages;
  uint4* my_q = reinterpret_cast<uint4*>(qs + warp * C::kQBytes);

  // ahead: the walk of the copies, its next page's id read one step early
  Walk ahead = rd;
  long long ua = u0;
  int next_id = c.table[(long long)ahead.t.r * c.row_pages + ahead.t.p0 + ahead.page];
  auto issue = [&](int stage) {
    const int id = next_id;
    const bool ok = id >= 0 && id < c.num_pages;
    if (lane == 0) {
      my_bad[stage] = !ok;
      if (ok) {
        mbar_arrive_expect_tx(&my_bar[stage], C::kBlock);
        bulk_g2s(my_ring + stage * C::kBlock, kv4_block(c, a.layer, id, ahead.head), C::kBlock, &my_bar[stage]);
      } else {
        set_status(c.status, JX_ERR_RANGE);
        mbar_arrive(&my_bar[stage]);
      }
    }
    if (++ua < u1) {
      ahead.next<C::kRows>(a);
      next_id = c.table[(long long)ahead.t.r * c.row_pages + ahead.t.p0 + ahead.page];
    }
  };
#pragma unroll
  for (int s = 0; s < C::kStages; ++s)
    if (ua < u1) issue(s);

  float acc[C::kMT][NT][4], m[NT][2], l[NT][2];
  int last[NT][2];                       // last visible key of the thread's columns (-1: none)
  uint4 q[C::kQReg ? NT : 1][C::kQReg ? C::kQParts : 1][C::kQReg ? HD / 32 : 1];
  bool fresh = true;
  int stage = 0;
  uint32_t phase = 0;

  for (long long u = u0; u < u1; ++u) {
    if (fresh) {
      fresh = false;
      const int f0 = rd.t.qt * C::kRows, F = a.S * a.G;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int f = f0 + nt * 8 + 2 * t + e, s = f / a.G;
          last[nt][e] = f < F && s < rd.t.cnt ? rd.t.base + s : -1;
          m[nt][e] = -INFINITY, l[nt][e] = 0.f;
        }
        const int f = f0 + nt * 8 + g, s = f / a.G;
        const bool live = f < F && s < rd.t.cnt;
        const T* src = static_cast<const T*>(a.q) + rd.t.r * a.q_row + s * a.q_tok +
                       (rd.head * a.G + (f - s * a.G)) * a.q_head;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          const int d = (i / C::kWords) * 128 + t * (C::kWords * 8) + (i % C::kWords) * 8;
          uint4 x[C::kQParts];
          if (live) {
            q_words(src + d, a.q_vec, x);
          } else {
#pragma unroll
            for (int p = 0; p < C::kQParts; ++p) x[p] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int p = 0; p < C::kQParts; ++p) {
            if constexpr (C::kQReg) q[nt][p][i] = x[p];
            else my_q[((nt * C::kQParts + p) * (HD / 32) + i) * 32 + lane] = x[p];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < C::kMT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][nt][e] = 0.f;
    }
    const bool arrived = mbar_wait_bounded(&my_bar[stage], phase);
    if (!__all_sync(~0u, arrived)) {      // give up: no copy of this warp may be in flight when it ends
      if (lane == 0) set_status(c.status, JX_ERR_TIMEOUT);
      for (int s = 0; s < C::kStages; ++s) mbar_wait_bounded(&my_bar[s], s < stage ? phase ^ 1 : phase);
      return;
    }
    const unsigned char* blk = my_ring + stage * C::kBlock;
    const int key0 = (rd.t.p0 + rd.page) * kPage;
    const int f_last = min(rd.t.qt * C::kRows + C::kRows, rd.t.cnt * a.G) - 1;
    const int pos0 = rd.t.base + rd.t.qt * C::kRows / a.G, pos1 = rd.t.base + f_last / a.G;
    // every key is seen by every row of the tile that is there
    const bool all = key0 + kPage - 1 <= pos0 && (a.window <= 0 || key0 > pos1 - a.window) &&
                     rd.t.qt * C::kRows + C::kRows <= rd.t.cnt * a.G;
    if (!my_bad[stage]) {
#pragma unroll
      for (int sub = 0; sub < kPage / C::kKeys; ++sub) {
        const int kb = sub * C::kKeys;
        float sc[kTiles][NT][4];
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[i][nt][e] = 0.f;
#pragma unroll
        for (int ch = 0; ch < C::kChunks; ++ch) {
          const int group = HD >= 128 ? ch * 4 + t : t >> 1;
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            uint32_t kw[2][C::kWords], s2[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = kb + i * 16 + h * 8 + g;
              const unsigned char* p = blk + key * (HD / 2) + ch * 64 + t * (C::kWords * 4);
              if constexpr (C::kWords == 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                kw[h][0] = x.x, kw[h][1] = x.y, kw[h][2] = x.z, kw[h][3] = x.w;
              } else {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                kw[h][0] = x.x, kw[h][1] = x.y;
              }
              s2[h] = lds16(blk + kPage * HD + (key * (HD / 32) + group) * 2) * 0x10001u;
            }
#pragma unroll
            for (int wd = 0; wd < C::kWords; ++wd) {
              uint32_t x[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < 4; ++k) x[h][k] = scaled(kw[h][wd], k, s2[h]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int p = 0; p < C::kQParts; ++p) {
                  uint4 b;
                  if constexpr (C::kQReg) b = q[nt][p][ch * C::kWords + wd];
                  else b = my_q[((nt * C::kQParts + p) * (HD / 32) + ch * C::kWords + wd) * 32 + lane];
                  mma_bf16(sc[i][nt], x[0][0], x[1][0], x[0][1], x[1][1], b.x, b.y);
                  mma_bf16(sc[i][nt], x[0][2], x[1][2], x[0][3], x[1][3], b.z, b.w);
                }
            }
          }
        }
        // softmax over the keys: registers (key g: 0, 1), (key g + 8: 2, 3) of columns 2t, 2t + 1
        uint32_t pf[kTiles][NT][C::kPParts][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float x = sc[i][nt][2 * h + e] * a.scale_log2;
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
            const float use = mx == -INFINITY ? 0.f : mx;      // nothing visible yet: every term is 2^-inf
            const float f = exp2_f(m[nt][e] - use);
            m[nt][e] = mx;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float x = exp2_f(sc[i][nt][2 * h + e] - use);
                sc[i][nt][2 * h + e] = x;
                sum += x;
              }
            l[nt][e] = l[nt][e] * f + sum;
            if (__any_sync(~0u, f != 1.f)) {      // seldom, once a row's maximum has settled
#pragma unroll
              for (int i = 0; i < C::kMT; ++i) acc[i][nt][e] *= f, acc[i][nt][2 + e] *= f;
            }
          }
#pragma unroll
          for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x0 = sc[i][nt][2 * h], x1 = sc[i][nt][2 * h + 1];
#pragma unroll
              for (int p = 0; p < C::kPParts; ++p) {
                // probabilities rounded to bfloat16 (2^-9) for bfloat16 results, split in three for float32 ones
                const uint32_t r = pack_bf16x2(x0, x1);
                pf[i][nt][p][h] = transpose8x8(r);
                if (p + 1 < C::kPParts) x0 -= rnd<bf16>(x0), x1 -= rnd<bf16>(x1);
              }
            }
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const int vg = HD == 64 ? g >> 2 : HD == 128 ? g >> 1 : g;   // the thread's channels are of one group
          uint32_t vw[4][C::kVWords], s2[2];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + i * 16 + 2 * t + (j & 1) + (j >> 1) * 8;
            const unsigned char* p = blk + kPage * (HD / 2) + key * (HD / 2) + g * (C::kVWords * 4);
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
          for (int h = 0; h < 2; ++h) {
            const unsigned char* p = blk + kPage * HD + kPage * (HD / 32) * 2 + ((kb + i * 16 + 2 * t + h * 8) * (HD / 32) + vg) * 2;
            uint32_t s = lds16(p) | (lds16(p + (HD / 32) * 2) << 16);
            // NaN and infinity to 0: a key that a row does not see has P = 0 there, and 0 * NaN would reach it.  Rows that
            // do see one get NaN below.
            const uint32_t zero = 0u, most = 0x7F7F7F7Fu;
            __nv_bfloat162 b = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&s), *reinterpret_cast<const __nv_bfloat162*>(&zero));
            b = __hmin2(b, *reinterpret_cast<const __nv_bfloat162*>(&most));
            s2[h] = *reinterpret_cast<uint32_t*>(&b);
          }
#pragma unroll
          for (int wd = 0; wd < C::kVWords; ++wd) {
            const uint32_t lo0 = __byte_perm(vw[0][wd], vw[1][wd], 0x5410), hi0 = __byte_perm(vw[0][wd], vw[1][wd], 0x7632);
            const uint32_t lo1 = __byte_perm(vw[2][wd], vw[3][wd], 0x5410), hi1 = __byte_perm(vw[2][wd], vw[3][wd], 0x7632);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a0 = scaled(lo0, k, s2[0]), a1 = scaled(hi0, k, s2[0]);
              const uint32_t a2 = scaled(lo1, k, s2[1]), a3 = scaled(hi1, k, s2[1]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int p = 0; p < C::kPParts; ++p)
                  mma_bf16(acc[wd * 4 + k][nt], a0, a1, a2, a3, pf[i][nt][p][0], pf[i][nt][p][1]);
            }
          }
        }
      }
      // a NaN scale of values: the rows that see its key get NaN in its channels
      constexpr int kV = kPage * (HD / 32) / 2;   // 32-bit words of value scales
      const uint32_t* vs = reinterpret_cast<const uint32_t*>(blk + kPage * HD + kPage * (HD / 32) * 2);
      bool nan = false;
#pragma unroll
      for (int i = 0; i < kV / 32; ++i) {
        const uint32_t x = vs[i * 32 + lane];
        nan |= (x & 0x7FFFu) >= 0x7F80u || (x & 0x7FFF0000u) >= 0x7F800000u;
      }
      if (__any_sync(~0u, nan)) {
        const int vg = HD == 64 ? g >> 2 : HD == 128 ? g >> 1 : g;
        for (int key = 0; key < kPage; ++key) {
          if ((lds16(reinterpret_cast<const unsigned char*>(vs) + (key * (HD / 32) + vg) * 2) & 0x7FFFu) < 0x7F80u) continue;
          const int at = key0 + key;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (at <= last[nt][e] && (a.window <= 0 || at > last[nt][e] - a.window)) {
#pragma unroll
                for (int i = 0; i < C::kMT; ++i) acc[i][nt][e] = acc[i][nt][2 + e] = __uint_as_float(0x7FC00000u);
              }
        }
        __syncwarp();
      }
    }
    __syncwarp();
    if (ua < u1) issue(stage);
    if (++stage == C::kStages) stage = 0, phase ^= 1;

    const bool seg_end = rd.page + 1 == rd.t.n;
    if (seg_end || u + 1 == u1) {
      const bool whole = seg_end && seg_first >= u0;
      const int f0 = rd.t.qt * C::kRows, F = a.S * a.G;
      float* slot = a.part + (w * 2 + (seg_first >= u0 ? 1 : 0)) * C::kSlot;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[nt][e];
          sum += __shfl_xor_sync(~0u, sum, 4);
          sum += __shfl_xor_sync(~0u, sum, 8);
          sum += __shfl_xor_sync(~0u, sum, 16);
          const int j = nt * 8 + 2 * t + e, f = f0 + j;
          if (f >= F) continue;
          if (whole) {
            const int s = f / a.G;
            T* o = static_cast<T*>(a.out) +
                   (((long long)rd.t.r * a.S + s) * a.Hq + rd.head * a.G + (f - s * a.G)) * HD + g * (C::kVWords * 8);
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int wd = 0; wd < C::kVWords; ++wd) {
              float x[8];
#pragma unroll
              for (int k = 0; k < 4; ++k) x[k] = acc[wd * 4 + k][nt][e] * inv, x[4 + k] = acc[wd * 4 + k][nt][2 + e] * inv;
              if constexpr (C::kF32) {
                reinterpret_cast<float4*>(o + wd * 8)[0] = make_float4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<float4*>(o + wd * 8)[1] = make_float4(x[4], x[5], x[6], x[7]);
              } else {
                *reinterpret_cast<uint4*>(o + wd * 8) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                                                   pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
              }
            }
          } else {
            float* o = slot + j * HD + g * (C::kVWords * 8);
#pragma unroll
            for (int wd = 0; wd < C::kVWords; ++wd) {
              *reinterpret_cast<float4*>(o + wd * 8) = make_float4(acc[wd * 4][nt][e], acc[wd * 4 + 1][nt][e],
                                                                   acc[wd * 4 + 2][nt][e], acc[wd * 4 + 3][nt][e]);
              *reinterpret_cast<float4*>(o + wd * 8 + 4) =
                  make_float4(acc[wd * 4][nt][2 + e], acc[wd * 4 + 1][nt][2 + e], acc[wd * 4 + 2][nt][2 + e],
                              acc[wd * 4 + 3][nt][2 + e]);
            }
            if (g == 0) slot[C::kRows * HD + 2 * j] = m[nt][e], slot[C::kRows * HD + 2 * j + 1] = sum;
          }
        }
    }
    if (u + 1 < u1) {
      if (seg_end) seg_first = u + 1, fresh = true;
      rd.next<C::kRows>(a);
    }
  }
}

// Joins what several warps hold of one (row, tile, head): a CTA for every query row of it.  Rows without a visible key are
// zero.
constexpr int kJoinWarps = 8;
template <int HD, typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_join_kernel(const AttendArgs a, int rows) {
  pdl_wait();
  __shared__ float sh[kJoinWarps][HD + 2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, Hkv = a.c.num_kv_heads;
  const long long seg = blockIdx.x;
  const long long item = seg / Hkv;
  const int head = (int)(seg - item * Hkv), j = blockIdx.y;
  const long long units = a.total[0], warps = a.total[1];
  const long long first = a.item_first[item], end = item + 1 < a.items ? a.item_first[item + 1] : units;
  const long long n = (end - first) / Hkv, u0 = first + head * n, u1 = u0 + n;
  const long long w0 = n ? run_of(u0, units, warps) : 0, w1 = n ? run_of(u1 - 1, units, warps) : 0;
  if (n && w0 == w1) return;
  const int r = (int)(item / a.tiles), qt = (int)(item - (long long)r * a.tiles), f = qt * rows + j, s = f / a.G;
  if (f >= a.S * a.G) return;
  T* out = static_cast<T*>(a.out) + (((long long)r * a.S + s) * a.Hq + head * a.G + (f - s * a.G)) * HD;
  const int slot_floats = rows * (HD + 2);
  constexpr int kV = HD / 32;
  float m = -INFINITY, l = 0.f, o[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) o[i] = 0.f;
  for (long long w = w0 + warp; n && w <= w1; w += kJoinWarps) {
    const float* slot = a.part + (w * 2 + (run_start(w, units, warps) <= u0 ? 1 : 0)) * slot_floats;
    const float mw = slot[rows * HD + 2 * j], lw = slot[rows * HD + 2 * j + 1];
    const float mn = fmaxf(m, mw), use = mn == -INFINITY ? 0.f : mn;
    const float fo = exp2_f(m - use), fw = exp2_f(mw - use);
    m = mn;
    l = l * fo + lw * fw;
#pragma unroll
    for (int i = 0; i < kV; ++i) o[i] = o[i] * fo + slot[j * HD + i * 32 + lane] * fw;
  }
#pragma unroll
  for (int i = 0; i < kV; ++i) sh[warp][i * 32 + lane] = o[i];
  if (lane == 0) sh[warp][HD] = m, sh[warp][HD + 1] = l;
  __syncthreads();
  float mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) mx = fmaxf(mx, sh[w][HD]);
  const float use = mx == -INFINITY ? 0.f : mx;
  float fw[kJoinWarps];
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) fw[w] = exp2_f(sh[w][HD] - use), sum += sh[w][HD + 1] * fw[w];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int d = tid; d < HD; d += kJoinWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) x += sh[w][d] * fw[w];
    out[d] = from_f<T>(x * inv);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------
// Query rows are taken in tiles of 8, 16 or 32: the smallest that holds all S * G rows of a KV head, or 32 (16 where the
// accumulators of 32 rows would not fit the registers), which then reads every page once per tile.
int n_tiles_of(int hd, int dtype, int rows) {
  const int most = hd == 256 || dtype == JX_F32 ? 2 : 4;
  return rows <= 8 ? 1 : rows <= 16 || most == 2 ? 2 : 4;
}

struct Layout {
  int nt, tiles;
  long long items, first_at, total_at, part_at, bytes;
};
int sm_count() {
  static int n[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!n[dev] && (cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n[dev] <= 0)) n[dev] = 148;
  return n[dev];
}
constexpr int kMostCtas = 160, kMostWarps = 8;
Layout layout_of(const jx_kv4_cache& c, int S, int Hq, int dtype) {
  Layout l;
  const int G = Hq / c.num_kv_heads;
  const long long rows = (long long)S * G;
  l.nt = n_tiles_of(c.head_dim, dtype, rows > 64 ? 64 : (int)rows);
  l.tiles = (int)((rows + 8 * l.nt - 1) / (8 * l.nt));
  l.items = (long long)c.num_rows * l.tiles;
  l.total_at = 0;
  l.first_at = 16;
  l.part_at = (l.first_at + l.items * 8 + 15) / 16 * 16;
  l.bytes = l.part_at + (long long)kMostCtas * kMostWarps * 2 * (8 * l.nt) * (c.head_dim + 2) * 4;
  return l;
}

template <int HD, int NT, typename T>
int launch(AttendArgs& a, cudaStream_t s) {
  using C = Cfg<HD, NT, T>;
  static_assert(C::kWarps <= kMostWarps, "workspace");
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(kv4_attend_kernel<HD, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
      return JX_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  const long long most = (long long)a.items * a.c.row_pages * a.c.num_kv_heads;   // units there can be
  int grid = sm_count() < kMostCtas ? sm_count() : kMostCtas;
  if (most < grid) grid = (int)most;
  kv4_attend_kernel<HD, NT, T><<<grid, C::kThreads, C::kSmem, s>>>(a);
  if (cudaPeekAtLastError() != cudaSuccess) return JX_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.items * (long long)a.c.num_kv_heads), (unsigned)(a.tiles > 1 || a.S * a.G >= 8 * NT ? 8 * NT : a.S * a.G));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<HD, T>, (const AttendArgs)a, C::kRows) == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

template <int HD, typename T>
int launch_nt(int nt, AttendArgs& a, cudaStream_t s) {
  if (nt == 1) return launch<HD, 1, T>(a, s);
  if constexpr (HD < 256 && sizeof(T) == 2)
    if (nt == 4) return launch<HD, 4, T>(a, s);
  return launch<HD, 2, T>(a, s);
}

template <typename T>
int launch_hd(int nt, AttendArgs& a, cudaStream_t s) {
  if (a.c.head_dim == 64) return launch_nt<64, T>(nt, a, s);
  if (a.c.head_dim == 128) return launch_nt<128, T>(nt, a, s);
  return launch_nt<256, T>(nt, a, s);
}

}  // namespace

long long kv4_attend_workspace(const jx_kv4_cache& c, int S, int Hq, int dtype) { return layout_of(c, S, Hq, dtype).bytes; }

int run_kv4_attend(const jx_kv4_cache& c, int layer, int S, int Hq, const void* q, const long long* qs, void* out,
                   float scale, int window, void* ws, int dtype, cudaStream_t s) {
  const Layout l = layout_of(c, S, Hq, dtype);
  AttendArgs a;
  a.c = c, a.layer = layer, a.S = S, a.Hq = Hq, a.G = Hq / c.num_kv_heads, a.window = window;
  a.items = (int)l.items, a.tiles = l.tiles, a.scale_log2 = scale * 1.4426950408889634f;
  a.q = q, a.q_row = qs[0], a.q_tok = qs[1], a.q_head = qs[2], a.out = out;
  const int unit = dtype == JX_BF16 ? 8 : 4;
  a.q_vec = !((uintptr_t)q & 15) && !(qs[0] % unit) && !(qs[1] % unit) && !(qs[2] % unit);
  unsigned char* b = static_cast<unsigned char*>(ws);
  a.total = reinterpret_cast<long long*>(b + l.total_at);
  a.item_first = reinterpret_cast<long long*>(b + l.first_at);
  a.part = reinterpret_cast<float*>(b + l.part_at);
  return dtype == JX_BF16 ? launch_hd<bf16>(l.nt, a, s) : launch_hd<float>(l.nt, a, s);
}

}  // namespace jxb
