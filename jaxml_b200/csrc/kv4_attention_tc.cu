// Attention of many query rows (prompt chunks, long drafts) over the 4-bit KV cache, on tcgen05.
//
// A CTA takes 128 query rows of one KV head (positions x the heads that share it) and a run of pages:
//   warps 4-7  turn a page's codes into bfloat16 operands in shared memory (exact: 4-bit code x 4-bit scale), K as
//              [64 keys][hd] and V transposed as [hd][64 keys], both K-major without swizzle, K a page ahead of V;
//   warps 0-3  own a query row each thread: scores out of TMEM, running maximum and sum, P back over the scores;
//   warp 8     issues S = Q K^T and O += P V, warp 9 the copies of the pages.
// S has two buffers, so the scores of the next page are made while this one's softmax runs: what is left in line is the
// softmax itself.  P is an A operand in TMEM, and so is Q where two S buffers, O and Q fit (not for hd 128 with two CTAs).
// What runs for every page is kept short (loops over halves, groups and pieces, not unrolled): 20 KB of instructions in turn
// on one multiprocessor were fetched again for every page, and that fetching was the bound.
// The maximum that the exponents refer to moves only when a score passes it by 2^8, so O in TMEM is rescaled a few times a
// row instead of every page, and l is summed in float32.  Probabilities are up to 2^8 then and round to bfloat16 anywhere in
// a binade, where with the true maximum the largest are 1 or just below it, the finest part of one: the rounding's part of a
// result's relative error is 0.0015 to 0.0017 instead of 0.0007 to 0.0009 (simulated, 4000 keys), 0.0022 in all for the chunk
// below where the mma.sync kernels have 0.0017.
// Two CTAs share a multiprocessor (256 TMEM columns each).
//
// Work is split as in kv4_attention.cu: all (row, tile, KV head, page) units cut into equal runs, one a CTA; parts of a
// (row, tile, head) meet in the join kernel.  What bounds it is the issue of instructions: a page and 128 rows take some
// 4000 of them a warp's width (codes to operands 1300, softmax 1000, the rest waits, walks and what a tile costs once), 1300
// cycles of a multiprocessor, where the 8192 exponentials and the products take 512 each.  Measured (B200): 2 rows of 512
// queries and 32 heads over 4096 and 2538 tokens of 8 heads of 128: 107 us, 470 TFLOP/s; 18 us for 1000 keys more, so some
// 30 us are the start, the change of tiles and the join.
#include "kv4_attend.cuh"

namespace jxb {
using namespace kv4;
namespace {

constexpr int kRows = 128, kSoft = 128, kDeq = 128, kThreads = kSoft + kDeq + 64, kRing = 3;

template <int kOff>
__device__ __forceinline__ uint32_t lds_u32(uint32_t at) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(r) : "r"(at), "n"(kOff));
  return r;
}
template <int kOff>
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) {
  uint16_t r;
  asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(r) : "r"(at), "n"(kOff));
  return r;
}
__device__ __forceinline__ void lds_v2(uint32_t at, uint32_t& a, uint32_t& b) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(at));
}
__device__ __forceinline__ void lds_v4(uint32_t at, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(at));
}
__device__ __forceinline__ void sts_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Keys 2 E and 2 E + 1 of a group of 8: a word of codes each, at `vp` and `other` bytes on (offsets of the group's first
// pair), and their scales as a pair, at `sp` of the group's first key.
template <int HD, int E>
__device__ __forceinline__ void load_keys(uint32_t vp, uint32_t other, uint32_t sp, uint32_t* x, uint32_t* sc) {
  constexpr int kLine = 2 * E * (HD / 2), kXor = (kLine >> 7 & (HD / 32 - 1)) << 4;
  const uint32_t at = vp ^ kXor;
  x[2 * E] = lds_u32<kLine>(at);
  // at head_dim 256 a key is a line of its own, and the other key of the pair has its last bit in the xor
  x[2 * E + 1] = lds_u32<kLine>((HD == 256 ? at ^ 16u : at) + other);
  constexpr int kKey = HD / 16, kPair = 2 * E * kKey, kHigh = kPair & ~15, kLow = kPair & 15;
  if constexpr (kKey == 16) sc[E] = lds_u16<0>(sp ^ kPair) | lds_u16<0>(sp ^ (kPair + 16)) << 16;
  else sc[E] = lds_u16<kLow>(sp ^ kHigh) | lds_u16<kLow + kKey>(sp ^ kHigh) << 16;
}

template <int HD>
struct Tc {
  static constexpr int kBlock = kPage * HD + kPage * (HD / 32) * 4;
  static constexpr bool kQTmem = HD != 128;
  static constexpr int kKBytes = kPage * HD * 2;
  static constexpr int kKSbo = HD / 8 * 128;            // between groups of 8 keys (or query rows)
  static constexpr int kVSbo = kPage / 8 * 128 + 16;    // between groups of 8 channels; 16 bytes off for the banks
  static constexpr int kVBytes = HD / 8 * kVSbo;
  static constexpr int kSCol = kQTmem ? HD / 2 : 0, kOCol = kSCol + 2 * kPage;
  static constexpr int kCols = kOCol + HD <= 256 ? 256 : 512;
  static constexpr int kCtas = kCols == 256 ? 2 : 1;
  static constexpr int kOffK = kRing * kBlock, kOffV = kOffK + kKBytes, kOffQ = kOffV + 2 * kVBytes;
  static constexpr int kOffBar = kOffQ + (kQTmem ? 0 : kRows * HD * 2);
  static constexpr int kOffNan = kOffBar + 16 * 8, kOffMisc = kOffNan + 2 * 8 * 8, kOffFirst = kOffMisc + 80;
  static constexpr int kUsed = kOffFirst + (kThreads + 40) * 8 + 1024;
  // no third CTA beside two of 256 columns: it would wait for TMEM
  static constexpr int kSmem = kCtas == 2 ? (kUsed > 80 * 1024 ? kUsed : 80 * 1024) : (kUsed > 116 * 1024 ? kUsed : 116 * 1024);
  static_assert(kSmem <= (kCtas == 2 ? 113 : 227) * 1024, "shared memory");
  static_assert(kOCol + HD <= 512, "TMEM");
  static_assert(kOffK % 16 == 0 && kOffV % 16 == 0 && kVBytes % 16 == 0 && kOffQ % 16 == 0, "alignment");
};

// D[tmem] (+)= A[tmem] * B[shared]
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 columns of 32-bit cells of the warp's 32 lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Scores outside [from, to] to -inf.
__device__ __forceinline__ void hide(uint32_t* x, int from, int to) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (k < from || k > to) x[k] = 0xFF800000u;
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two floats at a time.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, Tc<HD>::kCtas)
    kv4_attend_tc_kernel(const AttendArgs a, const __grid_constant__ CUtensorMap map) {
  using C = Tc<HD>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* kbuf = smem + C::kOffK;
  unsigned char* vbuf = smem + C::kOffV;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t *page_full = bar, *page_free = bar + 3, *v_ready = bar + 6, *s_done = bar + 8, *pv_done = bar + 10, *k_ready = bar + 12,
           *p_ready = bar + 13, *q_ready = bar + 14;
  unsigned char* nan_keys = smem + C::kOffNan;          // [2][8 groups][8 bytes]: keys of the page with a NaN value scale
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* bad = reinterpret_cast<int*>(tmem_slot + 2);     // [8]: whether pages i, i + 1, ... have no block
  int* last = bad + 8;                                  // [8]: whether they end a segment
  long long* first = reinterpret_cast<long long*>(smem + C::kOffFirst);
  long long* sums = first + kThreads + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const jx_kv4_cache& c = a.c;

  if (tid == 0) {
    prefetch_tmap(&map);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&page_full[i], 1);
      mbar_init(&page_free[i], kDeq / 32);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_ready[i], kDeq / 32);
      mbar_init(&s_done[i], 1);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(k_ready, kDeq / 32);
    mbar_init(p_ready, kSoft / 32);
    mbar_init(q_ready, kSoft / 32);
    *dead = 0;
    fence_barrier_init();
  }
  if (warp == 4) {
    tmem_alloc(tmem_slot, C::kCols);
    tmem_relinquish();
  }
  // units before each thread's share of the items, and all of them
  const int each = (a.items + kThreads - 1) / kThreads;
  const int i0 = min(a.items, tid * each), i1 = min(a.items, i0 + each);
  long long mine = 0;
  for (int i = i0; i < i1; ++i) mine += (long long)item_at<kRows>(a, i).n * c.num_kv_heads;
  long long v = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) sums[warp] = v;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();   // the join's launch is under way; it waits for this kernel's end
  const uint32_t tmem = *tmem_slot;
  long long before = 0, units = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    units += sums[w];
  }
  first[tid] = before + v - mine;
  const long long runs = min((long long)gridDim.x, max(units, 1ll));
  if (blockIdx.x == 0) {
    long long u = before + v - mine;
    for (int i = i0; i < i1; ++i) {
      a.item_first[i] = u;
      if (c.counts[i / a.tiles] > a.S) set_status(c.status, JX_ERR_RANGE);
      u += (long long)item_at<kRows>(a, i).n * c.num_kv_heads;
    }
    if (tid == 0) a.total[0] = units, a.total[1] = runs;
  }
  __syncthreads();

  const long long w = blockIdx.x;
  const bool work = units > 0 && w < runs;
  if (work) {
    const long long u0 = run_start(w, units, runs), u1 = run_start(w + 1, units, runs);
    Walk at;
    {
      int lo = 0, hi = kThreads - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= u0) lo = mid;
        else hi = mid - 1;
      }
      long long u = first[lo];
      at.item = (long long)lo * each;
      while (true) {
        at.t = item_at<kRows>(a, at.item);
        const long long n = (long long)at.t.n * c.num_kv_heads;
        if (u0 < u + n) break;
        u += n;
        ++at.item;
      }
      at.head = (int)((u0 - u) / at.t.n);
      at.page = (int)((u0 - u) - (long long)at.head * at.t.n);
    }
    // every wait is bounded; once one has run out all roles leave
    auto wait = [&](uint64_t* b, uint32_t parity) {
      if (try_wait_long(b, parity)) return true;
      const long long t0 = clock64();
      while (!try_wait_long(b, parity)) {
        if (*dead) return false;
        if (clock64() - t0 > kWaitCycles) {
          *dead = 1;
          set_status(c.status, JX_ERR_TIMEOUT);
          return false;
        }
      }
      return true;
    };

    // the warp's writes stand: one arrival
    auto arrive = [&](uint64_t* b) {
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };

    if (warp >= 8) {
      const int pages = (int)(u1 - u0);
      if (warp == 8 && lane == 0) {
        // ---------------- products ----------------
        constexpr uint32_t kIdS = umma_idesc_bf16_f32(128, kPage), kIdO = umma_idesc_bf16_f32(128, HD);
        const uint64_t kd = umma_desc_kmajor(smem_u32(kbuf), 128, C::kKSbo);
        const uint64_t qd = umma_desc_kmajor(smem_u32(smem + C::kOffQ), 128, C::kKSbo);
        uint32_t qp = 0;
        auto scores = [&](int i, bool start) {
          // K, Q of a new segment, and the page before last is through with this S buffer
          const int b = i & 1;
          if (!wait(k_ready, i & 1) || (start && !wait(q_ready, qp)) || (i >= 2 && !wait(&pv_done[b], ((i - 2) >> 1) & 1)))
            return false;
          qp ^= start;
          tc_fence_after();
          const uint32_t sd = tmem + C::kSCol + b * kPage;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            if constexpr (C::kQTmem) umma_ts(sd, tmem + kk * 8, kd + (uint64_t)(kk * 16), kIdS, kk > 0);
            else umma_bf16(sd, qd + (uint64_t)(kk * 16), kd + (uint64_t)(kk * 16), kIdS, kk > 0);
          }
          umma_commit(&s_done[b]);
          return true;
        };
        bool ok = scores(0, true), fresh = true;
        for (int i = 0; i < pages && ok; ++i) {
          const int b = i & 1;
          const bool next = i + 1 < pages, start = last[i & 7];   // page i + 1 begins a segment
          // its scores first, unless they wait for a Q that follows the results of this page
          if (next && !start && !(ok = scores(i + 1, false))) break;
          ok = wait(&v_ready[b], (i >> 1) & 1) && wait(p_ready, i & 1);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = umma_desc_kmajor(smem_u32(vbuf + b * C::kVBytes), 128, C::kVSbo);
#pragma unroll
          for (int kk = 0; kk < kPage / 16; ++kk)
            umma_ts(tmem + C::kOCol, tmem + C::kSCol + b * kPage + kk * 8, vd + (uint64_t)(kk * 16), kIdO, !fresh || kk > 0);
          umma_commit(&pv_done[b]);
          fresh = start;
          if (next && start) ok = scores(i + 1, true);
        }
      } else if (warp == 9 && lane == 0) {
        // ---------------- copies ----------------
        int i = 0;
        for (; i < pages; ++i) {
          const int st = i % kRing;
          const int id = c.table[(long long)at.t.r * c.row_pages + at.t.p0 + at.page];
          if (i >= kRing && !wait(&page_free[st], (i / kRing - 1) & 1)) break;
          last[i & 7] = at.page + 1 == at.t.n;
          fetch<HD>(a, &map, id, at.head, smem + st * C::kBlock, &page_full[st], &bad[i & 7]);
          if (i + 1 < pages) at.next<kRows>(a);
        }
      }
      __syncwarp();
    } else if (warp >= 4) {
      // ---------------- pages to bfloat16 operands ----------------
      const int dt = tid - kSoft, dw = warp - 4;
      const int g = lane & 7, t4 = lane >> 3;
      const int pages = (int)(u1 - u0);
      // What a thread reads of a block, as offsets that the pages share.  The swizzle exchanges 16-byte pieces within 128
      // bytes by the number of the line, and blocks begin on whole lines: pieces are stepped through by xor.
      // K: lane (key g of a group of 8, word t4 of a 16-byte piece); a core matrix's rows are 8 neighbouring lanes
      const uint32_t ring = smem_u32(smem);
      const uint32_t k_codes = swz<HD>((dw * 16 + g) * (HD / 2)) + t4 * 4;
      const uint32_t k_to = smem_u32(kbuf) + dw * 2 * C::kKSbo + t4 * 128 + g * 16;
      // V: 8 keys x 8 channels (word ch of each key); half of a warp takes the keys of a pair the other way round, for the
      // banks
      constexpr int kVStep = kDeq / (HD / 8);      // groups of 8 keys that the threads cover at once
      const int ch = dt % (HD / 8), vj = dt / (HD / 8);
      const uint32_t flip = (lane >> 4) & 1;
      const uint32_t v_codes = swz<HD>(kPage * (HD / 2) + (vj * 8 + flip) * (HD / 2) + ch * 4);
      const uint32_t v_other = flip ? 0u - HD / 2 : HD / 2;
      // step i: K of page i, V of page i - 1
      int st = 0, ring_use = 0, last_st = 0;
      for (int i = 0; i <= pages; ++i) {
        if (i < pages) {
          const bool ok = wait(&page_full[st], ring_use) && (i == 0 || wait(&s_done[(i - 1) & 1], ((i - 1) >> 1) & 1));
          if (!__all_sync(~0u, ok)) break;
          const uint32_t blk = ring + st * C::kBlock;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const uint32_t sp = blk + swz<HD>(kPage * HD + ((dw * 2 + h) * 8 + g) * (HD / 16));
            uint32_t ks[HD / 64];        // the key's scales, two groups a register
            if constexpr (HD == 64) ks[0] = lds_u32<0>(sp);
            else if constexpr (HD == 128) lds_v2(sp, ks[0], ks[1]);
            else lds_v4(sp, ks[0], ks[1], ks[2], ks[3]);
            const uint32_t codes = blk + k_codes + h * (8 * (HD / 2)), to = k_to + h * C::kKSbo;
#pragma unroll
            for (int grp = 0; grp < HD / 32; ++grp) {
              const uint32_t x = lds_u32<0>(codes ^ (grp * 16));
              const uint32_t s2 = __byte_perm(ks[grp >> 1], 0, grp & 1 ? 0x3232 : 0x1010), c2 = minus136(s2);
              sts_v4(to + grp * 512, scaled2(x, 0, s2, c2), scaled2(x, 1, s2, c2), scaled2(x, 2, s2, c2), scaled2(x, 3, s2, c2));
            }
          }
          fence_proxy_async();
          arrive(k_ready);
        }
        if (i > 0) {
          const int j0 = i - 1, b = j0 & 1;
          const bool ok = j0 < 2 || wait(&pv_done[b], ((j0 - 2) >> 1) & 1);
          if (!__all_sync(~0u, ok)) break;
          const uint32_t blk = ring + last_st * C::kBlock, vd = smem_u32(vbuf) + b * C::kVBytes;
          constexpr int kBlocks = HD / 8 * (kPage / 8);
#pragma unroll 1
          for (int n = 0; n < (kBlocks + kDeq - 1) / kDeq; ++n) {
            const int j = vj + n * kVStep;
            if (kBlocks >= kDeq || dt < kBlocks) {
              // transposed in registers.  Keys 2 e and 2 e + 1 (exchanged where flip is set): their line's number adds an xor
              uint32_t x[8], sc[4], cc[4];
              const uint32_t vp = blk + v_codes + n * (kVStep * 8 * (HD / 2));
              const uint32_t sp = blk + swz<HD>(kPage * HD + kPage * (HD / 16) + j * 8 * (HD / 16) + (ch >> 2) * 2);
              load_keys<HD, 0>(vp, v_other, sp, x, sc);
              load_keys<HD, 1>(vp, v_other, sp, x, sc);
              load_keys<HD, 2>(vp, v_other, sp, x, sc);
              load_keys<HD, 3>(vp, v_other, sp, x, sc);
              uint32_t worst = 0;
#pragma unroll
              for (int e = 0; e < 4; ++e) worst |= bad_scales(sc[e]);
              uint32_t nans = 0;
              if (worst & 0x80008000u) {
                // no scale of the format: 0 for the product (0 * NaN would reach rows that do not see the key), noted for
                // those that do
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t bad2 = bad_scales(sc[e]);
                  if (bad2 & 0x8000u) sc[e] &= 0xFFFF0000u, nans |= 1u << (2 * e);
                  if (bad2 & 0x80000000u) sc[e] &= 0x0000FFFFu, nans |= 2u << (2 * e);
                }
              }
              if ((ch & 3) == 0) nan_keys[(b * 8 + (ch >> 2)) * 8 + j] = (unsigned char)nans;
              const uint32_t lo_sel = flip ? 0x1054u : 0x5410u, hi_sel = flip ? 0x3276u : 0x7632u;
              const uint32_t to = vd + ch * C::kVSbo + j * 128;
              uint32_t lo[4], hi[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                cc[e] = minus136(sc[e]);
                lo[e] = __byte_perm(x[2 * e], x[2 * e + 1], lo_sel);
                hi[e] = __byte_perm(x[2 * e], x[2 * e + 1], hi_sel);
              }
#pragma unroll 1
              for (int k = 0; k < 4; ++k) {
                uint32_t r[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  r[e] = scaled2(lo[e], 0, sc[e], cc[e]), r[4 + e] = scaled2(hi[e], 0, sc[e], cc[e]);
                  lo[e] >>= 4, hi[e] >>= 4;
                }
                sts_v4(to + k * 16, r[0], r[1], r[2], r[3]);
                sts_v4(to + (k + 4) * 16, r[4], r[5], r[6], r[7]);
              }
            }
          }
          fence_proxy_async();
          arrive(&v_ready[b]);
          arrive(&page_free[last_st]);
        }
        last_st = st;
        if (++st == kRing) st = 0, ring_use ^= 1;
      }
    } else {
      // ---------------- softmax: one query row a thread ----------------
      const uint32_t mine_at = tmem + ((uint32_t)(warp * 32) << 16);
      const float c2 = a.scale_log2;
      long long seg_first = u0 - at.page;
      bool start = true;
      float m = -INFINITY, l = 0.f;
      int hi = -1, lo = 0, all_hi = -1, all_lo = -1, f = 0;
      uint32_t nan_groups = 0;
      int i = 0;
      for (long long u = u0; u < u1; ++u, ++i) {
        const int b = i & 1;
        const uint32_t use = (i >> 1) & 1, s_at = mine_at + C::kSCol + b * kPage;
        if (start) {
          start = false;
          const int f0 = at.t.qt * kRows, F = a.S * a.G;
          f = f0 + tid;
          const int s = f / a.G;
          const bool live = f < F && s < at.t.cnt;
          hi = live ? at.t.base + s : -1;
          lo = live && a.window > 0 ? max(0, hi - a.window + 1) : 0;
          // what rows that are not there make of a page does not matter: zeros are written for them
          all_hi = at.t.base + f0 / a.G;
          all_lo = a.window > 0 ? at.t.base + (f0 + kRows - 1) / a.G - a.window : -1;
          m = -INFINITY, l = 0.f, nan_groups = 0;
          const bf16* src = static_cast<const bf16*>(a.q) + at.t.r * a.q_row + s * a.q_tok + (at.head * a.G + (f - s * a.G)) * a.q_head;
#pragma unroll 1
          for (int part = 0; part < HD / 64; ++part) {
            uint32_t r[32];
            QPiece<bf16> piece[8];
            q_load<8>(src + part * 64, 8, live, a.q_vec, piece);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              uint4 x;
              q_words(piece[k], a.sign, &x);
              r[4 * k] = x.x, r[4 * k + 1] = x.y, r[4 * k + 2] = x.z, r[4 * k + 3] = x.w;
            }
            __syncwarp();
            if constexpr (C::kQTmem) {
              tmem_st32(mine_at + part * 32, r);
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                *reinterpret_cast<uint4*>(smem + C::kOffQ + (tid >> 3) * C::kKSbo + (part * 8 + k) * 128 + (tid & 7) * 16) =
                    make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
            }
          }
          if constexpr (C::kQTmem) {
            tmem_wait_st();
            tc_fence_before();
          } else {
            fence_proxy_async();
          }
          arrive(q_ready);
        }
        bool ok = wait(&s_done[b], use);
        if (!__all_sync(~0u, ok)) break;
        tc_fence_after();
        const int key0 = (at.t.p0 + at.page) * kPage;
        const bool all = key0 + kPage - 1 <= all_hi && key0 > all_lo && !bad[i & 7];
        const int from = bad[i & 7] ? kPage : lo - key0, to = hi - key0;      // the row sees keys [from, to] of the page
        float mx = -INFINITY;
#pragma unroll 1
        for (int h = 0; h < 64; h += 32) {
          uint32_t x[32];
          tmem_ld32(s_at + h, x);
          tmem_wait_ld();
          if (!all) hide(x, from - h, to - h);
          float mz = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
#pragma unroll
          for (int k = 2; k < 32; k += 4) {
            mx = max3(mx, __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
            if (k + 2 < 32) mz = max3(mz, __uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
          }
          mx = fmaxf(mx, mz);
        }
        const bool moves = (mx - m) * c2 > 8.f;           // also from -inf, when there is nothing to rescale
        const bool scales = moves && m != -INFINITY;
        if (__any_sync(~0u, scales)) {
          ok = i == 0 || wait(&pv_done[b ^ 1], ((i - 1) >> 1) & 1);
          if (!__all_sync(~0u, ok)) break;
          tc_fence_after();
          const float fo = scales ? exp2_f((m - mx) * c2) : 1.f;
          l *= fo;
#pragma unroll 1
          for (int part = 0; part < HD / 32; ++part) {
            uint32_t r[32];
            tmem_ld32(mine_at + C::kOCol + part * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * fo);
            tmem_st32(mine_at + C::kOCol + part * 32, r);
          }
          tmem_wait_st();
        }
        if (moves) m = mx;
        const float ref = m == -INFINITY ? 0.f : -m * c2;
        uint64_t sum2 = pair(0.f, 0.f);
        const uint64_t c22 = pair(c2, c2), ref2 = pair(ref, ref);
#pragma unroll 1
        for (int h = 0; h < 64; h += 32) {
          uint32_t x[32];
          tmem_ld32(s_at + h, x);
          tmem_wait_ld();
          if (!all) hide(x, from - h, to - h);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float p0, p1;
            unpair(fma2(pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), c22, ref2), p0, p1);
            p0 = exp2_f(p0), p1 = exp2_f(p1);
            sum2 = add2(sum2, pair(p0, p1));
            x[k] = pack_bf16x2(p0, p1);       // probabilities in bfloat16: half a step, 2^-9 of their binade's top
          }
          tmem_st16(s_at + h / 2, x);         // over scores that have been read
        }
        float s0, s1;
        unpair(sum2, s0, s1);
        l += s0 + s1;
        tmem_wait_st();
        tc_fence_before();
        ok = wait(&v_ready[b], use);
        if (!__all_sync(~0u, ok)) break;
        {
          const unsigned long long* nk = reinterpret_cast<const unsigned long long*>(nan_keys + b * 64);
          unsigned long long any = 0;
#pragma unroll
          for (int grp = 0; grp < HD / 32; ++grp) any |= nk[grp];
          if (any && !bad[i & 7]) {
            const int from = max(lo - key0, 0), to = min(hi - key0, kPage - 1);
            if (from <= to) {
              const unsigned long long sees = (~0ull << from) & (~0ull >> (63 - to));
              for (int grp = 0; grp < HD / 32; ++grp)
                if (nk[grp] & sees) nan_groups |= 1u << grp;
            }
          }
        }
        arrive(p_ready);
        const bool seg_end = at.page + 1 == at.t.n;
        if (seg_end || u + 1 == u1) {
          ok = wait(&pv_done[b], use);
          if (!__all_sync(~0u, ok)) break;
          tc_fence_after();
          const bool whole = seg_end && seg_first >= u0, there = f < a.S * a.G;
          float* slot = a.part + (w * 2 + (seg_first >= u0 ? 1 : 0)) * (long long)(kRows * (HD + 2));
          if (hi < 0) m = -INFINITY, l = 0.f;               // padding
          const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
          bf16* o = there ? out_row<HD, bf16>(a, at.t.r, at.head, f) : nullptr;
#pragma unroll 1
          for (int part = 0; part < HD / 32; ++part) {
            uint32_t r[32];
            tmem_ld32(mine_at + C::kOCol + part * 32, r);
            tmem_wait_ld();
            if (there) {
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  y[e] = hi < 0 ? 0.f        // padding: a visible key of NaN makes its O NaN, which times 0 stays
                         : (nan_groups >> part) & 1u ? __uint_as_float(0x7FC00000u) : __uint_as_float(r[k + e]) * inv;
                if (whole) store_row8<bf16>(o + part * 32 + k, y);
                else
#pragma unroll
                  for (int e = 0; e < 8; e += 4)
                    *reinterpret_cast<float4*>(slot + ((part * 32 + k + e) / 4 * kRows + tid) * 4) =
                        make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
              }
            }
            __syncwarp();
          }
          if (!whole && there) slot[kRows * HD + 2 * tid] = m * c2, slot[kRows * HD + 2 * tid + 1] = l;
          tc_fence_before();
        }
        if (u + 1 < u1) {
          if (seg_end) seg_first = u + 1, start = true;
          at.next<kRows>(a);
        }
      }
    }
  }
  // after a wait that ran out: what was issued gets as long again to finish before its memory goes
  __syncthreads();
  if (*dead && tid == 0) {
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitCycles) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
}

template <int HD>
int launch(const AttendArgs& a, const CUtensorMap& map, int sms, cudaStream_t s) {
  using C = Tc<HD>;
  static bool ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return JX_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    if (cudaFuncSetAttribute(kv4_attend_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
      return JX_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  kv4_attend_tc_kernel<HD><<<sms * C::kCtas, kThreads, C::kSmem, s>>>(a, map);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

}  // namespace

int run_kv4_attend_tc(const void* args, const void* map, int sms, cudaStream_t s) {
  const AttendArgs& a = *static_cast<const AttendArgs*>(args);
  const CUtensorMap& m = *static_cast<const CUtensorMap*>(map);
  if (a.c.head_dim == 64) return launch<64>(a, m, sms, s);
  if (a.c.head_dim == 128) return launch<128>(a, m, sms, s);
  return launch<256>(a, m, sms, s);
}

}  // namespace jxb
