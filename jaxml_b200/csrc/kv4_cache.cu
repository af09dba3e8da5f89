// Writing, reading back and managing the pages of the 4-bit KV cache (format in kv4.cuh).
//
// Rows own pages through a table [rows][row_pages] of page ids (-1: none) shared by all layers; refs counts the
// rows that hold a page.  Forked rows share pages; a shared page that is not full is copied when a row is about to
// write on it (copy on write in jx_kv4_extend).  Every choice of a page is the lowest free one, rows in order, so the
// same calls give the same tables whatever the scheduling; the only atomics are integer counts.
#include "kv4.cuh"

namespace jxb {
namespace {

// ------------------------------------------------------------------------------------------------
// append: one CTA per token; 8 channels a thread, 4 threads a group
// ------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float* x);
template <>
__device__ __forceinline__ void load8<bf16>(const bf16* p, bool vec, float* x) {
  if (vec) {
    unpack8(*reinterpret_cast<const uint4*>(p), x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(p[i]);
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, bool vec, float* x) {
  if (vec) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}

struct AppendArgs {
  jx_kv4_cache c;
  int layer, S, vec;
  const void* src[2];
  long long row[2], tok[2], head[2];   // element strides
};

// The nibbles of 8 values of a group.  bfloat16 values: the quotient by a product with 1 / s and one step of correction,
// which is the correctly rounded one where that matters: a quotient that is a half step is represented exactly, so the
// correction lands on it, and any other is off a half step by at least 2^-9 of itself, far beyond what the step leaves.
// float32 values, and scales near the ends of the range, take the division.
template <typename T>
__device__ __forceinline__ uint32_t nibbles(const float* x, float s) {
  uint32_t w = 0;
  if (sizeof(T) == 2 && s > 1e-30f && s < 1e30f) {
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q0 = x[j] * inv, q = fmaf(fmaf(-q0, s, x[j]), inv, q0);
      // 1.5 * 2^23 + q rounds to an integer (ties to even) in the lower bits; + 8 makes the nibble.  |q| <= 7.44: no clamp
      w |= (__float_as_uint(q + 12582920.f) & 15u) << (4 * j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w |= kv4_nibble(x[j], s) << (4 * j);
  }
  return w;
}

// Each CTA takes kTok neighbouring tokens of a row: their loads are under way together.
template <typename T, int kTok>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  const jx_kv4_cache& c = a.c;
  const int hd = c.head_dim, per = hd >> 3, items = 2 * c.num_kv_heads * per, tiles = (a.S + kTok - 1) / kTok;
  for (long long t = blockIdx.x; t < (long long)c.num_rows * tiles; t += gridDim.x) {
    const int r = (int)(t / tiles), i0 = (int)(t - (long long)r * tiles) * kTok;
    const int cnt = c.counts[r];
    if (i0 == 0 && cnt > a.S && threadIdx.x == 0) set_status(c.status, JX_ERR_RANGE);
    if (i0 >= cnt) continue;
    const int pos0 = c.lengths[r] - cnt + i0;
    int page[kTok];
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      const int pos = pos0 + j;
      page[j] = -1;
      if (i0 + j < min(cnt, a.S)) {
        if (pos >= 0 && pos < c.row_pages * kPage) page[j] = c.table[(long long)r * c.row_pages + pos / kPage];
        if (page[j] < 0 || page[j] >= c.num_pages) {
          page[j] = -1;
          if (threadIdx.x == 0) set_status(c.status, JX_ERR_RANGE);
        }
      }
    }
    for (int it = threadIdx.x; it < items; it += blockDim.x) {   // items and blockDim are multiples of 4
      const int which = it >= items / 2, rest = it - which * (items / 2), head = rest / per, ch = rest % per;
      const T* p = static_cast<const T*>(a.src[which]) + r * a.row[which] + i0 * a.tok[which] +
                   head * a.head[which] + ch * 8;
      float x[kTok][8];
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        if (page[j] >= 0) {
          load8<T>(p + j * a.tok[which], a.vec, x[j]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[j][e] = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[j][e]) & 0x7FFFFFFFu);
        const unsigned group = 0xFu << (threadIdx.x & 28);
        m = max(m, __shfl_xor_sync(group, m, 1));
        m = max(m, __shfl_xor_sync(group, m, 2));
        if (page[j] < 0) continue;
        const float s = kv4_scale(m);
        const int slot = (pos0 + j) % kPage;
        unsigned char* blk = kv4_block(c, a.layer, page[j], head);
        *reinterpret_cast<uint32_t*>(blk + which * kPage * (hd / 2) + slot * (hd / 2) + ch * 4) = nibbles<T>(x[j], s);
        if ((ch & 3) == 0)
          *reinterpret_cast<bf16*>(blk + kv4_scale_offset(hd, which) + (slot * (hd / 32) + (ch >> 2)) * 2) =
              __float2bfloat16_rn(s);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// read back: token start + i of every row, zeros outside it
// ------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x);
template <>
__device__ __forceinline__ void store8<bf16>(bf16* p, const float* x) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                            pack_bf16x2(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float* x) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

template <typename T, int kTok>
__global__ void __launch_bounds__(256) kv4_read_kernel(const jx_kv4_cache c, int layer, const int* start, int start_add, int n,
                                                       T* k, T* v) {
  const int hd = c.head_dim, per = hd >> 3, items = 2 * c.num_kv_heads * per, tiles = (n + kTok - 1) / kTok;
  for (long long t = blockIdx.x; t < (long long)c.num_rows * tiles; t += gridDim.x) {
    const int r = (int)(t / tiles), i0 = (int)(t - (long long)r * tiles) * kTok;
    const long long pos0 = (long long)(start ? start[r] : 0) + start_add + i0;
    const int len = min(c.lengths[r], c.row_pages * kPage);
    int page[kTok];
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      page[j] = -1;
      if (pos0 + j >= 0 && pos0 + j < len) {
        page[j] = c.table[(long long)r * c.row_pages + (pos0 + j) / kPage];
        if (page[j] < 0 || page[j] >= c.num_pages) {
          page[j] = -1;
          if (threadIdx.x == 0 && i0 + j < n) set_status(c.status, JX_ERR_RANGE);
        }
      }
    }
    for (int it = threadIdx.x; it < items; it += blockDim.x) {
      const int which = it >= items / 2, rest = it - which * (items / 2), head = rest / per, ch = rest % per;
      uint32_t w[kTok];
      float s[kTok];
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        w[j] = 0x88888888u, s[j] = 0.f;
        if (page[j] >= 0) {
          const unsigned char* blk = kv4_block(c, layer, page[j], head);
          const int slot = (int)((pos0 + j) & (kPage - 1));
          w[j] = *reinterpret_cast<const uint32_t*>(blk + which * kPage * (hd / 2) + slot * (hd / 2) + ch * 4);
          s[j] = to_f(*reinterpret_cast<const bf16*>(blk + kv4_scale_offset(hd, which) + (slot * (hd / 32) + (ch >> 2)) * 2));
        }
      }
#pragma unroll
      for (int j = 0; j < kTok; ++j) {
        if (i0 + j >= n) continue;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)((int)((w[j] >> (4 * e)) & 15u) - 8) * s[j];
        store8<T>((which ? v : k) + ((((long long)r * n + i0 + j) * c.num_kv_heads + head) * hd + ch * 8), x);
      }
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
  const int len = c.lengths[r], cut = rows ? len : (n ? n[r] : n_all), held = min(pages_of(max(len, 0)), c.row_pages);
  __syncthreads();
  if (cut < 0 || cut > len) {
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
  const int items = 2 * c.num_kv_heads * (c.head_dim / 8);
  const int threads = items < 256 ? (items + 31) / 32 * 32 : 256;
  const int tok = S >= 4 ? 4 : 1;
  const long long tiles = (long long)c.num_rows * ((S + tok - 1) / tok);
  const int grid = (int)(tiles < 148 * 64 ? tiles : 148 * 64);
  if (dtype == JX_BF16) {
    if (tok == 4) kv4_append_kernel<bf16, 4><<<grid, threads, 0, s>>>(a);
    else kv4_append_kernel<bf16, 1><<<grid, threads, 0, s>>>(a);
  } else {
    if (tok == 4) kv4_append_kernel<float, 4><<<grid, threads, 0, s>>>(a);
    else kv4_append_kernel<float, 1><<<grid, threads, 0, s>>>(a);
  }
  return cudaPeekAtLastError() == cudaSuccess ? JX_OK : JX_ERR_CUDA;
}

int run_kv4_read(const jx_kv4_cache& c, int layer, const int* start, int start_add, int n, void* k, void* v, int dtype,
                 cudaStream_t s) {
  const int items = 2 * c.num_kv_heads * (c.head_dim / 8);
  const int threads = items < 256 ? (items + 31) / 32 * 32 : 256;
  const int tok = n >= 4 ? 4 : 1;
  const long long tiles = (long long)c.num_rows * ((n + tok - 1) / tok);
  const int grid = (int)(tiles < 148 * 64 ? tiles : 148 * 64);
  if (dtype == JX_BF16) {
    if (tok == 4) kv4_read_kernel<bf16, 4><<<grid, threads, 0, s>>>(c, layer, start, start_add, n, (bf16*)k, (bf16*)v);
    else kv4_read_kernel<bf16, 1><<<grid, threads, 0, s>>>(c, layer, start, start_add, n, (bf16*)k, (bf16*)v);
  } else {
    if (tok == 4) kv4_read_kernel<float, 4><<<grid, threads, 0, s>>>(c, layer, start, start_add, n, (float*)k, (float*)v);
    else kv4_read_kernel<float, 1><<<grid, threads, 0, s>>>(c, layer, start, start_add, n, (float*)k, (float*)v);
  }
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
