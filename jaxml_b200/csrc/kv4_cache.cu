// Writing, reading back and managing the pages of the 4-bit KV cache (format in kv4.cuh).
//
// Rows own pages through a table [rows][row_pages] of page ids (-1: none) shared by all layers; refs counts the
// rows that hold a page.  Forked rows share pages; a shared page that is not full is copied when a row is about to
// write on it (copy on write in jx_kv4_extend).  Every choice of a page is the lowest free one, rows in order, so the
// same calls give the same tables whatever the scheduling; the only atomics are integer counts.
#include <algorithm>

#include "kv4.cuh"

namespace jxb {
namespace {

// ------------------------------------------------------------------------------------------------
// append and read.  A thread owns 8 channels of one head of keys or values (4 threads a group of 32) and goes through
// tiles of kTok neighbouring positions: a tile starts at a multiple of kTok, so it lies in one page, and its loads are
// under way together.  The tile's scales are 32 neighbouring bytes at 128 channels; thread j of a group handles the
// j-th token's.  What bounds a large call is instructions, about as many as its bytes allow (100 a warp and 8 values a
// thread to write, 80 to read).  Measured (B200): 16 rows of up to 512 tokens, 8 heads of 128, bf16: written and read back
// in 17 us, 4.0 TB/s of what both have to move; one token a row of 64: 4.6 us.
// ------------------------------------------------------------------------------------------------
template <typename T>
struct Eight;   // 8 values as they lie in memory
template <>
struct Eight<bf16> {
  uint4 v;
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const bf16* p, bool vec) {
    if (vec) {
      v = *reinterpret_cast<const uint4*>(p);
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
      v = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16,
                     q[6] | (uint32_t)q[7] << 16);
    }
  }
  __device__ __forceinline__ uint32_t amax_bits() const {   // two 16-bit maxima at a time, widened at the end
    uint32_t m = max_u16x2(max_u16x2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), max_u16x2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
    return max(m & 0xFFFF0000u, m << 16);
  }
  static __device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ void get(float* x) const { unpack8(v, x); }
};
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p, bool vec) {
    if (vec) {
      a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    } else {
      a = make_float4(p[0], p[1], p[2], p[3]), b = make_float4(p[4], p[5], p[6], p[7]);
    }
  }
  __device__ __forceinline__ void get(float* x) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  __device__ __forceinline__ uint32_t amax_bits() const {
    float x[8];
    get(x);
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
    return m;
  }
};

struct AppendArgs {
  jx_kv4_cache c;
  int layer, S, vec;
  const void* src[2];
  long long row[2], tok[2], head[2];   // element strides
};

// The nibbles of 8 values of a group.  bfloat16 values x = X 2^a (X <= 255) over a scale s = M 2^b (M <= 15): a quotient
// that is no half step is off each of them by at least 1 / 30 or by a 255th of itself, 2^-10.  So x times an approximate
// 1 / s (off by 2^-19 at most), added to 6144 and rounded there to a multiple of 2^-11, is a half step exactly where x / s
// is one, and the second sum rounds it to an integer, ties to even, leaving 8 + q in its low byte.  |q| <= 7.44: no clamp.
// float32 values, and scales near the ends of the range, take the division.
template <typename T>
__device__ __forceinline__ uint32_t nibbles(const Eight<T>& v, float s) {
  float x[8];
  v.get(x);
  uint32_t w = 0;
  if (sizeof(T) == 2 && s > 1e-30f && s < 1e30f) {
    float inv;
    asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s));
    uint32_t n[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = __float_as_uint(fmaf(x[j], inv, 6144.f) + (12582920.f - 6144.f));
    const uint32_t even = __byte_perm(__byte_perm(n[0], n[2], 0x0040), __byte_perm(n[4], n[6], 0x0040), 0x5410);
    const uint32_t odd = __byte_perm(__byte_perm(n[1], n[3], 0x0040), __byte_perm(n[5], n[7], 0x0040), 0x5410);
    w = odd * 16u + even;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w |= kv4_nibble(x[j], s) << (4 * j);
  }
  return w;
}

template <typename T, int HD, int kTok>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  static_assert(kTok == 1 || kTok == 4, "a group of four threads shares the scales of four tokens");
  const jx_kv4_cache& c = a.c;
  constexpr int kPer = HD / 8;
  const int it = blockIdx.y * blockDim.x + threadIdx.x, half = c.num_kv_heads * kPer;
  const int tiles = (a.S + kTok - 1) / kTok + (kTok > 1), lane = threadIdx.x & 31;
  const bool lead = it == 0, live = it < 2 * half;   // the others only take part in the shuffles
  const int which = live && it >= half, head = live ? (it - which * half) / kPer : 0, ch = it % kPer;
  const T* src = static_cast<const T*>(a.src[which]) + head * a.head[which] + ch * 8;
  const long long tok = a.tok[which];
  // a cache made of given tensors may hold any length: first is kept where sums with positions do not wrap, and so that no
  // position below the row's end is another's
  const int r = blockIdx.z, cnt = max(c.counts[r], 0), n = min(cnt, a.S);
  const int first = min(max(c.lengths[r], 0) - cnt, c.row_pages * kPage);
  if (lead && blockIdx.x == 0 && cnt > a.S) set_status(c.status, JX_ERR_RANGE);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int base = (first & ~(kTok - 1)) + tile * kTok, i0 = base - first;   // tokens i0 .. i0 + kTok - 1 of n
    if (i0 >= n) break;
    if (i0 + kTok <= 0) continue;
    int page = -1;
    if (base >= 0 && base < c.row_pages * kPage) page = c.table[(long long)r * c.row_pages + base / kPage];
    if (page < 0 || page >= c.num_pages) {
      if (lead) set_status(c.status, JX_ERR_RANGE);
      continue;
    }
    const T* p = src + r * a.row[which] + i0 * tok;
    Eight<T> x[kTok];
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      if (live && i0 + j >= 0 && i0 + j < n) x[j].load(p + j * tok, a.vec);
      else x[j].zero();
    }
    uint32_t own = 0;
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      uint32_t m = x[j].amax_bits();
      m = max(m, __shfl_xor_sync(~0u, m, 1));
      m = max(m, __shfl_xor_sync(~0u, m, 2));
      if (kTok == 1 || (lane & 3) == j) own = m;
    }
    const float scale = kv4_scale(own);
    const int slot = base % kPage;
    unsigned char* blk = kv4_block(c, a.layer, page, head);
    unsigned char* at = blk + (which * kPage + slot) * (HD / 2) + ch * 4;
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      const float s = kTok == 1 ? scale : __shfl_sync(~0u, scale, j, 4);
      if (live && i0 + j >= 0 && i0 + j < n) *reinterpret_cast<uint32_t*>(at + j * (HD / 2)) = nibbles<T>(x[j], s);
    }
    const int mine = kTok == 1 ? 0 : lane & 3;
    if (live && (kTok == 1 ? (lane & 3) == 0 : i0 + mine >= 0 && i0 + mine < n))
      *reinterpret_cast<bf16*>(blk + kv4_scale_offset(HD, which) + ((slot + mine) * (HD / 32) + (ch >> 2)) * 2) =
          __float2bfloat16_rn(scale);
  }
}

// Read back: token start + i of every row, zeros outside it.
__device__ __forceinline__ void store8(bf16* p, uint4 v) { *reinterpret_cast<uint4*>(p) = v; }
__device__ __forceinline__ void store8(float* p, uint4 v) {
  float x[8];
  unpack8(v, x);
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

template <typename T, int HD, int kTok>
__global__ void __launch_bounds__(256) kv4_read_kernel(const jx_kv4_cache c, int layer, const int* start, int start_add, int n,
                                                       T* k, T* v) {
  constexpr int kPer = HD / 8;
  const int it = blockIdx.y * blockDim.x + threadIdx.x, half = c.num_kv_heads * kPer;
  const int tiles = (n + kTok - 1) / kTok + (kTok > 1);
  const int which = it >= half, head = (it - which * half) / kPer, ch = it % kPer;
  T* dst = (which ? v : k) + (long long)head * HD + ch * 8;
  const long long tok = (long long)c.num_kv_heads * HD;
  if (it >= 2 * half) return;
  const int r = blockIdx.z, len = min(c.lengths[r], c.row_pages * kPage);
  const long long first = (long long)(start ? start[r] : 0) + start_add;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long base = (first & ~(long long)(kTok - 1)) + (long long)tile * kTok;
    const int i0 = (int)(base - first);
    if (i0 >= n) break;
    if (i0 + kTok <= 0) continue;
    int page = -1;
    if (base >= 0 && base < len) {
      page = c.table[(long long)r * c.row_pages + base / kPage];
      if (page < 0 || page >= c.num_pages) {
        page = -1;
        if (it == 0) set_status(c.status, JX_ERR_RANGE);
      }
    }
    uint32_t w[kTok], s[kTok];
#pragma unroll
    for (int j = 0; j < kTok; ++j) w[j] = 0x88888888u, s[j] = 0;
    if (page >= 0) {
      const unsigned char* blk = kv4_block(c, layer, page, head);
      const int slot = (int)(base & (kPage - 1));
      const unsigned char* at = blk + (which * kPage + slot) * (HD / 2) + ch * 4;
      const unsigned char* sc = blk + kv4_scale_offset(HD, which) + (slot * (HD / 32) + (ch >> 2)) * 2;
#pragma unroll
      for (int j = 0; j < kTok; ++j)
        if (base + j < len) {
          w[j] = *reinterpret_cast<const uint32_t*>(at + j * (HD / 2));
          s[j] = *reinterpret_cast<const uint16_t*>(sc + j * (HD / 32) * 2);
        }
    }
    T* out = dst + ((long long)r * n + i0) * tok;
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      if (i0 + j < 0 || i0 + j >= n) continue;
      uint4 o;
      if (s[j] < kKv4BadScale) {
        // (128 + u) s - 136 s (kv4.cuh), for the nibbles e and e + 4 at a time
        const uint32_t s2 = s[j] * 0x10001u, c2 = kv4::minus136(s2);
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = kv4::scaled2(w[j], e, s2, c2);
        o = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410), __byte_perm(x[0], x[1], 0x7632),
                       __byte_perm(x[2], x[3], 0x7632));
      } else {   // NaN, or no scale of this format
        float x[8];
        const float f = __uint_as_float(s[j] << 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)((int)((w[j] >> (4 * e)) & 15u) - 8) * f;
        o = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
      }
      store8(out + j * tok, o);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// page management
// ------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// Exclusive sum over the block's threads; *total gets the whole sum.  Every thread calls it.
__device__ __forceinline__ int block_exclusive(int x, int* sh /* [33] */, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();   // sh may still be read from an earlier call
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  if (warp == 0) {
    const int n = blockDim.x >> 5;
    int w = lane < n ? sh[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(~0u, w, d);
      if (lane >= d) w += o;
    }
    sh[lane] = w;
  }
  __syncthreads();
  *total = sh[(blockDim.x >> 5) - 1];
  return v - x + (warp ? sh[warp - 1] : 0);
}

// Workspace (ints): [0] page copies, [4, 4 + 2 * max(rows, pages)) their (source, destination), then [pages] free
// list or new ids, [rows] pages needed, [rows] shared page written on.
struct Plan {
  int* n;
  int* pair;
  int* list;
  int* need;
  int* part;
};
__host__ __device__ __forceinline__ Plan plan_of(int* ws, int rows, int pages) {
  const long long most = rows > pages ? rows : pages;
  Plan p;
  p.n = ws;
  p.pair = ws + 4;
  p.list = p.pair + 2 * most;
  p.need = p.list + pages;
  p.part = p.need + rows;
  return p;
}

// Rows [first, last) of a contiguous share of n items for this thread.
__device__ __forceinline__ void share_of(int n, int* first, int* last) {
  const int each = (n + (int)blockDim.x - 1) / (int)blockDim.x;
  *first = min(n, (int)threadIdx.x * each);
  *last = min(n, *first + each);
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPage - 1) / kPage; }

// One CTA: what each row needs, the lowest free pages in row order, tables and counts.  All or nothing: where a row
// would pass its table or the pool has too few pages, the status word is set and nothing but counts (zero) changes.
__global__ void __launch_bounds__(kPlanThreads) kv4_extend_plan_kernel(const jx_kv4_cache c, const int* counts,
                                                                       int count, int* ws) {
  __shared__ int sh[33];
  __shared__ int bad, copies;
  const int tid = threadIdx.x, R = c.num_rows, N = c.num_pages;
  const Plan p = plan_of(ws, R, N);
  if (tid == 0) bad = 0, copies = 0;
  __syncthreads();
  // the last page of a row that goes on inside it
  for (int r = tid; r < R; r += kPlanThreads) {
    const int len = c.lengths[r], cnt = counts ? counts[r] : count;
    int part = -1;
    if (len < 0 || cnt < 0 || (long long)len + cnt > (long long)c.row_pages * kPage) {
      bad = 1;
    } else if (cnt > 0 && len % kPage) {
      part = c.table[(long long)r * c.row_pages + len / kPage];
      if (part < 0 || part >= N) bad = 1, part = -1;
    }
    p.part[r] = part;
  }
  __syncthreads();
  int need = 0, first = 0, last = 0;
  if (!bad) {
    // a shared page is copied by every row that writes on it but its last holder
    share_of(R, &first, &last);
    for (int r = first; r < last; ++r) {
      const int len = c.lengths[r], cnt = counts ? counts[r] : count, part = p.part[r];
      int mine = cnt > 0 ? pages_of(len + cnt) - pages_of(len) : 0;
      if (part >= 0) {
        const int held = c.refs[part];
        if (held > 1) {
          int before = 0;
          for (int o = 0; o < r; ++o) before += p.part[o] == part;
          mine += held - before > 1;
        }
      }
      p.need[r] = mine;
      need += mine;
    }
  }
  int total, have = 0, free_before, free_total;
  int off = block_exclusive(need, sh, &total);
  if (total > 0) {   // the first `total` free pages, ascending
    int a, b;
    share_of(N, &a, &b);
    for (int i = a; i < b; ++i) have += c.refs[i] == 0;
    free_before = block_exclusive(have, sh, &free_total);
    for (int i = a; i < b && free_before < total; ++i)
      if (c.refs[i] == 0) p.list[free_before++] = i;
    if (tid == 0 && free_total < total) bad = 1;
  }
  __syncthreads();
  if (bad) {
    for (int r = tid; r < R; r += kPlanThreads) c.counts[r] = 0;
    if (tid == 0) {
      *p.n = 0;
      set_status(c.status, JX_ERR_RANGE);
    }
    return;
  }
  for (int r = first; r < last; ++r) {   // need becomes the row's first entry of the list
    const int mine = p.need[r];
    p.need[r] = off;
    off += mine;
  }
  __syncthreads();
  const int lane = tid & 31;
  for (int r = tid >> 5; r < R; r += kPlanThreads / 32) {
    const int len = c.lengths[r], cnt = counts ? counts[r] : count;
    const int at = pages_of(len), fresh = cnt > 0 ? pages_of(len + cnt) - at : 0;
    const int base = p.need[r], end = r + 1 < R ? p.need[r + 1] : total;
    const int copy = end - base - fresh;
    __syncwarp();     // counts may be the cache's own counts or lengths: all lanes have read them before lane 0 writes
    int* row = c.table + (long long)r * c.row_pages;
    for (int j = lane; j < fresh; j += 32) {
      const int page = p.list[base + copy + j];
      row[at + j] = page;
      c.refs[page] = 1;
    }
    if (lane == 0) {
      if (copy) {
        const int to = p.list[base], from = p.part[r], slot = atomicAdd(&copies, 1);
        p.pair[2 * slot] = from;
        p.pair[2 * slot + 1] = to;
        row[len / kPage] = to;
        c.refs[to] = 1;
        atomicSub(&c.refs[from], 1);
      }
      c.lengths[r] = len + cnt;
      c.counts[r] = cnt;
    }
    __syncwarp();
  }
  __syncthreads();
  if (tid == 0) *p.n = copies;
}

// One CTA: the used pages at or above the number of used pages move to the free ones below it, both ascending.
__global__ void __launch_bounds__(kPlanThreads) kv4_compact_plan_kernel(const jx_kv4_cache c, int* used_out, int* ws) {
  __shared__ int sh[33];
  const int tid = threadIdx.x, N = c.num_pages;
  const Plan p = plan_of(ws, c.num_rows, N);
  int a, b, used = 0, total;
  share_of(N, &a, &b);
  for (int i = a; i < b; ++i) used += c.refs[i] != 0;
  block_exclusive(used, sh, &total);
  int movers = 0, moves, holes = 0, n_holes;
  for (int i = a; i < b; ++i) movers += i >= total && c.refs[i] != 0, holes += i < total && c.refs[i] == 0;
  int m = block_exclusive(movers, sh, &moves), h = block_exclusive(holes, sh, &n_holes);
  for (int i = a; i < b; ++i) {
    const bool live = c.refs[i] != 0;
    if (i >= total && live) p.pair[2 * m++] = i;
    if (i < total && !live) p.pair[2 * h++ + 1] = i;
    p.list[i] = i;
  }
  __syncthreads();
  for (int k = tid; k < moves; k += kPlanThreads) {
    const int from = p.pair[2 * k], to = p.pair[2 * k + 1];
    p.list[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (tid == 0) {
    *p.n = moves;
    *used_out = total;
  }
}

// Bound by the bytes: 302 MB of pages moved in 90.5 us, 6.67 TB/s of reading and writing.
// Copies the planned pages (a page is one run of `bytes` in every layer); with `renumber`, table entries take their new
// ids first.  Sources and destinations are disjoint.
__global__ void __launch_bounds__(256) kv4_copy_pages_kernel(const jx_kv4_cache c, int* ws, long long bytes,
                                                             int renumber) {
  const Plan p = plan_of(ws, c.num_rows, c.num_pages);
  const int n = *p.n;
  if (n == 0) return;
  const long long stride = (long long)gridDim.x * blockDim.x, me = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (renumber)
    for (long long i = me; i < (long long)c.num_rows * c.row_pages; i += stride) {
      const int id = c.table[i];
      if (id >= 0 && id < c.num_pages) c.table[i] = p.list[id];
    }
  constexpr int kChunk = 256 * 16 * 2;
  const long long chunks = (bytes + kChunk - 1) / kChunk, work = (long long)n * c.num_layers * chunks;
  for (long long w = blockIdx.x; w < work; w += gridDim.x) {
    const long long pl = w / chunks, ch = w - pl * chunks;
    const int k = (int)(pl / c.num_layers), layer = (int)(pl - (long long)k * c.num_layers);
    const unsigned char* src = c.pages + ((long long)layer * c.num_pages + p.pair[2 * k]) * bytes;
    unsigned char* dst = c.pages + ((long long)layer * c.num_pages + p.pair[2 * k + 1]) * bytes;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long at = ch * kChunk + (j * 256 + threadIdx.x) * 16;
      if (at < bytes) *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(src + at);
    }
  }
}

// A column block of the table for all rows: read whole, then written from the parents' entries.
constexpr int kForkInts = 12288;
__global__ void __launch_bounds__(256) kv4_fork_kernel(const jx_kv4_cache c, const int* parents, int cols) {
  extern __shared__ int tile[];
  const int R = c.num_rows, P = c.row_pages, c0 = blockIdx.x * cols, w = min(cols, P - c0);
  for (int i = threadIdx.x; i < R * w; i += blockDim.x) tile[i] = c.table[(long long)(i / w) * P + c0 + i % w];
  __syncthreads();
  for (int i = threadIdx.x; i < R * w; i += blockDim.x) {
    const int r = i / w, j = i % w, from = parents[r];
    if (from >= R || from == r) continue;          // out of range: the row stays as it was (status below)
    const int old = tile[i], now = from < 0 ? -1 : tile[from * w + j];
    if (old == now) continue;
    c.table[(long long)r * P + c0 + j] = now;
    if (old >= 0 && old < c.num_pages) atomicSub(&c.refs[old], 1);
    if (now >= 0 && now < c.num_pages) atomicAdd(&c.refs[now], 1);
  }
  if (blockIdx.x == 0) {
    __syncthreads();
    for (int r = threadIdx.x; r < R; r += blockDim.x) tile[r] = c.lengths[r];
    __syncthreads();
    for (int r = threadIdx.x; r < R; r += blockDim.x) {
      const int from = parents[r];
      if (from >= R) set_status(c.status, JX_ERR_RANGE);
      else c.lengths[r] = from < 0 ? 0 : tile[from];
      c.counts[r] = 0;
    }
  }
}

// Rows named by the mask are emptied; without a mask every row loses its last n tokens.
__global__ void __launch_bounds__(128) kv4_shorten_kernel(const jx_kv4_cache c, const unsigned char* rows, const int* n,
                                                          int n_all) {
  const int r = blockIdx.x;
  if (rows && !rows[r]) return;
  // a length that no row can have (a cache made of given tensors) is only emptied: pages_of wraps near 2^31
  const int len = c.lengths[r], cut = rows ? len : (n ? n[r] : n_all), most = c.row_pages * kPage;
  const int held = pages_of(min(max(len, 0), most));
  __syncthreads();
  if (cut < 0 || cut > len || (len > most && cut < len)) {
    if (threadIdx.x == 0) {
      c.counts[r] = 0;
      set_status(c.status, JX_ERR_RANGE);
    }
    return;
  }
  int* row = c.table + (long long)r * c.row_pages;
  for (int j = pages_of(len - cut) + threadIdx.x; j < held; j += blockDim.x) {
    const int page = row[j];
    row[j] = -1;
    if (page >= 0 && page < c.num_pages) atomicSub(&c.refs[page], 1);
  }
  if (threadIdx.x == 0) {
    c.lengths[r] = len - cut;
    c.counts[r] = 0;
  }
}

// Tiles of four positions where single ones would fill the GPU's threads already: 8 channels a thread, 16 rows of 8 heads of
// 128 take 4.5 us a call with single positions and 5.2 with tiles at 4 tokens, 4.75 and 5.15 at 32, 6.8 and 6.2 at 64, 26.9
// and 16.9 at 512 (append and read).
bool tiles_of_four(const jx_kv4_cache& c, int n) {
  return n >= 4 && (long long)c.num_rows * n * 2 * c.num_kv_heads * (c.head_dim / 8) >= 1 << 18;
}

struct Shape {
  dim3 grid;
  int threads;
};
Shape shape_of(const jx_kv4_cache& c, int n, int tok) {
  const int items = 2 * c.num_kv_heads * (c.head_dim / 8), threads = items < 256 ? (items + 31) / 32 * 32 : 256;
  const int chunks = (items + threads - 1) / threads;
  const int tiles = (n + tok - 1) / tok + (tok > 1), most = std::max(1, 148 * 64 / (chunks * c.num_rows));
  return {dim3((unsigned)std::min(tiles, most), (unsigned)chunks, (unsigned)c.num_rows), threads};
}

template <typename T, int HD>
void launch_append_hd(const AppendArgs& a, cudaStream_t s) {
  if (tiles_of_four(a.c, a.S)) {
    const Shape g = shape_of(a.c, a.S, 4);
    kv4_append_kernel<T, HD, 4><<<g.grid, g.threads, 0, s>>>(a);
  } else {
    const Shape g = shape_of(a.c, a.S, 1);
    kv4_append_kernel<T, HD, 1><<<g.grid, g.threads, 0, s>>>(a);
  }
}
template <typename T>
void launch_append(const AppendArgs& a, cudaStream_t s) {
  if (a.c.head_dim == 64) launch_append_hd<T, 64>(a, s);
  else if (a.c.head_dim == 128) launch_append_hd<T, 128>(a, s);
  else launch_append_hd<T, 256>(a, s);
}

template <typename T, int HD>
void launch_read_hd(const jx_kv4_cache& c, int layer, const int* start, int start_add, int n, T* k, T* v, cudaStream_t s) {
  if (tiles_of_four(c, n)) {
    const Shape g = shape_of(c, n, 4);
    kv4_read_kernel<T, HD, 4><<<g.grid, g.threads, 0, s>>>(c, layer, start, start_add, n, k, v);
  } else {
    const Shape g = shape_of(c, n, 1);
    kv4_read_kernel<T, HD, 1><<<g.grid, g.threads, 0, s>>>(c, layer, start, start_add, n, k, v);
  }
}
template <typename T>
void launch_read(const jx_kv4_cache& c, int layer, const int* start, int start_add, int n, T* k, T* v, cudaStream_t s) {
  if (c.head_dim == 64) launch_read_hd<T, 64>(c, layer, start, start_add, n, k, v, s);
  else if (c.head_dim == 128) launch_read_hd<T, 128>(c, layer, start, start_add, n, k, v, s);
  else launch_read_hd<T, 256>(c, layer, start, start_add, n, k, v, s);
}

}  // namespace

int run_kv4_append(const jx_kv4_cache& c, int layer, int S, const void* k, const void* v, const long long* ks,
                   const long long* vs, int dtype, cudaStream_t s) {
  AppendArgs a;
  a.c = c, a.layer = layer, a.S = S;
  a.src[0] = k, a.src[1] = v;
  a.row[0] = ks[0], a.tok[0] = ks[1], a.head[0] = ks[2];
  a.row[1] = vs[0], a.tok[1] = vs[1], a.head[1] = vs[2];
  const int unit = dtype == JX_BF16 ? 8 : 4;   // elements in 16 bytes
  a.vec = 1;
  for (int i = 0; i < 2; ++i)
    if (((uintptr_t)a.src[i] & 15) || a.row[i] % unit || a.tok[i] % unit || a.head[i] % unit) a.vec = 0;
  if (dtype == JX_BF16) launch_append<bf16>(a, s);
  else launch_append<float>(a, s);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

int run_kv4_read(const jx_kv4_cache& c, int layer, const int* start, int start_add, int n, void* k, void* v, int dtype,
                 cudaStream_t s) {
  if (dtype == JX_BF16) launch_read(c, layer, start, start_add, n, (bf16*)k, (bf16*)v, s);
  else launch_read(c, layer, start, start_add, n, (float*)k, (float*)v, s);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

long long kv4_workspace_ints(int rows, int pages) {
  const long long most = rows > pages ? rows : pages;
  return 4 + 2 * most + pages + 2ll * rows;
}

static void copy_pages(const jx_kv4_cache& c, int* ws, int renumber, cudaStream_t s) {
  kv4_copy_pages_kernel<<<148 * 8, 256, 0, s>>>(c, ws, (long long)c.num_kv_heads * kv4_block_bytes(c.head_dim), renumber);
}

int run_kv4_extend(const jx_kv4_cache& c, const int* counts, int count, int* ws, cudaStream_t s) {
  kv4_extend_plan_kernel<<<1, kPlanThreads, 0, s>>>(c, counts, count, ws);
  copy_pages(c, ws, 0, s);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

int run_kv4_compact(const jx_kv4_cache& c, int* used, int* ws, cudaStream_t s) {
  kv4_compact_plan_kernel<<<1, kPlanThreads, 0, s>>>(c, used, ws);
  copy_pages(c, ws, 1, s);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

int run_kv4_fork(const jx_kv4_cache& c, const int* parents, cudaStream_t s) {
  int cols = kForkInts / c.num_rows;
  if (cols > c.row_pages) cols = c.row_pages;
  if (cols > 32) cols = 32;
  const int ints = c.num_rows * cols;
  kv4_fork_kernel<<<(c.row_pages + cols - 1) / cols, 256, ints * sizeof(int), s>>>(c, parents, cols);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

int run_kv4_shorten(const jx_kv4_cache& c, const unsigned char* rows, const int* n, int n_all, cudaStream_t s) {
  kv4_shorten_kernel<<<c.num_rows, 128, 0, s>>>(c, rows, n, n_all);
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

}  // namespace jxb
