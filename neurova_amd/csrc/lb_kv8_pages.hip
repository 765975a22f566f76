// The pages of the 8-bit cache: which row of a table holds which, how many rows hold
// each, and copies of them in every layer.
//
// A page is free when no row holds it, and free pages are handed out lowest first, so
// results depend on the state alone.  A row of `len` tokens holds the first
// ceil(len / page) entries of its table row.  Only these operators write a page's
// holders; everything stays on the GPU.
//
// Bound by latency: a few dependent loads (rows, lengths, holders, pages) and the
// launches.  free takes 2 to 5 us, fork 3 to 5, extend 8 to 11 (200 rows, and 100000 tokens
// for each of six; 200 rows with caches of 1, 32 and 64 layers and nothing to copy 9.7, 10.2
// and 11.4), the plan of compact 7 to 8.  One workgroup plans, since every count goes by all
// rows before it.  Copies are bound by HBM (951 pages of 128 KB in each of four layers, read
// and written: 190 us, 5.2 TB/s).
#include "attn_common.hpp"

namespace lb {
namespace {

struct Pages {
  int32_t *table, *lens, *refs;
  int64_t stride;
  int rows, width, pages, shift;  // shift: log2 of a page's tokens
};

// Rows of one call: a workgroup goes through all of them.
constexpr int kMaxRows = 4096;
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / kWave;
constexpr int kEach = kMaxRows / kPlanThreads;
// Rows of a table in which a row's first mention is found by its number, not by a search (extend
// of 4096 rows, of 4096 and of 9000: 16 and 296 us).
constexpr int kClaims = 8192;

// Pages of `tokens` (not below 0).
__device__ __forceinline__ int pages_of(int tokens, const Pages& p) { return (int)(((uint32_t)tokens + (1u << p.shift) - 1) >> p.shift); }
__device__ __forceinline__ int64_t capacity(const Pages& p) { return (int64_t)p.width << p.shift; }

// Exclusive prefix sum over the workgroup's threads; `total` of all.
__device__ __forceinline__ int block_scan(int v, int* lds, int& total) {
  const int upto = wave_scan(v), wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (lane == kWave - 1) lds[wave] = upto;
  __syncthreads();
  const int mine = lane < kPlanWaves ? lds[lane] : 0, before = wave_scan(mine);
  total = __builtin_amdgcn_readlane(before, kPlanWaves - 1);
  const int base = wave ? __builtin_amdgcn_readlane(before, wave - 1) : 0;
  __syncthreads();
  return base + upto - v;
}

// ------------------------------------------------------------------ free ---

// Entries of a table row that a workgroup goes through, one a thread and turn (with eight in
// turn: six rows of up to 1564 pages cut and extended 20.0 us and not 14.0).
constexpr int kCols = 256, kMostCols = 4096;
unsigned col_blocks(int64_t width) {
  const int64_t n = (width + kCols - 1) / kCols;
  return (unsigned)(n < 1 ? 1 : n < kMostCols ? n : kMostCols);
}

__global__ __launch_bounds__(256) void free_kernel(Pages p, const int32_t* rows, const int32_t* keep) {
  const int i = blockIdx.x, row = rows[i];
  if ((unsigned)row >= (unsigned)p.rows) return;
  const int tokens = keep ? max(keep[i], 0) : 0;
  const int first = pages_of(tokens, p);
  int32_t* mine = p.table + (int64_t)row * p.stride;
  for (int c = blockIdx.y * kCols + threadIdx.x; c < p.width; c += gridDim.y * kCols) {
    if (c < first || mine[c] < 0) continue;
    // a row that is named twice gives a page up once
    const int page = __hip_atomic_exchange(mine + c, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if ((unsigned)page < (unsigned)p.pages) __hip_atomic_fetch_add(p.refs + page, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (blockIdx.y == 0 && threadIdx.x == 0) __hip_atomic_fetch_min(p.lens + row, tokens, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ------------------------------------------------------------------ fork ---

// Tokens that request i gives its child; -1 if it is refused (a row outside the
// table, a child that holds tokens, or that an earlier request names).
__device__ __forceinline__ int forked(const Pages& p, const int32_t* parents, const int32_t* children, const int32_t* lens, int i, bool named) {
  const int parent = parents[i], child = children[i];
  if ((unsigned)parent >= (unsigned)p.rows || (unsigned)child >= (unsigned)p.rows || named || p.lens[child] > 0) return -1;
  int n = min(max(p.lens[parent], 0), lens ? max(lens[i], 0) : 0x7fffffff);
  return (int)min((int64_t)n, capacity(p));
}

__global__ __launch_bounds__(256) void fork_kernel(Pages p, const int32_t* parents, const int32_t* children, const int32_t* lens) {
  const int i = blockIdx.x, child = children[i];
  bool named = false;
  for (int j = threadIdx.x; j < i; j += 256) named |= children[j] == child;
  const int n = forked(p, parents, children, lens, i, __syncthreads_or(named));
  if (n <= 0) return;
  const int32_t* from = p.table + (int64_t)parents[i] * p.stride;
  int32_t* to = p.table + (int64_t)child * p.stride;
  const int last = pages_of(n, p);
  for (int c = blockIdx.y * kCols + threadIdx.x; c < last; c += gridDim.y * kCols) {
    const int page = from[c];
    const bool real = (unsigned)page < (unsigned)p.pages;
    to[c] = real ? page : -1;
    if (real) __hip_atomic_fetch_add(p.refs + page, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// The children's lengths, once their tables are written (which goes by the old ones).  TABLES:
// those as well, of up to kForkEntries entries in all, so that one launch does (together with
// the call that frees the children: 8 of 16 pages 5.5 us and not 6.9, 96 of 20 pages 7.6 and
// not 8.4; but 64 of 64 pages 8.8 and 8.7, 512 of 16 pages 30.7 and 18.1).
constexpr int kForkEach = 2, kForkEntries = kForkEach * kPlanThreads;
template <bool TABLES>
__global__ __launch_bounds__(kPlanThreads) void fork_lens_kernel(Pages p, const int32_t* parents, const int32_t* children, const int32_t* lens,
                                                                int32_t* done, int count) {
  __shared__ int32_t names[kMaxRows], claims[kClaims];
  int n[kEach];
  const bool few = p.rows <= kClaims;
  for (int i = threadIdx.x; i < count; i += kPlanThreads) {
    names[i] = children[i];
    if (few && (unsigned)names[i] < (unsigned)p.rows) claims[names[i]] = 0x7fffffff;
  }
  __syncthreads();
  if (few)
    for (int i = threadIdx.x; i < count; i += kPlanThreads)
      if ((unsigned)names[i] < (unsigned)p.rows) atomicMin(&claims[names[i]], i);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kPlanThreads + threadIdx.x;
    n[e] = -1;
    if (i >= count || (unsigned)names[i] >= (unsigned)p.rows) continue;
    bool named = false;
    if (few) named = claims[names[i]] != i;
    else
      for (int j = 0; j < i; ++j) named |= names[j] == names[i];
    n[e] = forked(p, parents, children, lens, i, named);
  }
  __syncthreads();
  if (TABLES) {
    int32_t* const tokens = claims;  // which are read no more
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (e * kPlanThreads + (int)threadIdx.x < count) tokens[e * kPlanThreads + threadIdx.x] = n[e];
    __syncthreads();
    int page[kForkEach], at[kForkEach];
#pragma unroll
    for (int e = 0; e < kForkEach; ++e) {
      const int x = e * kPlanThreads + threadIdx.x, i = x / max(p.width, 1), c = x - i * p.width;
      page[e] = -1, at[e] = -1;
      if (i >= count || c >= pages_of(max(tokens[i], 0), p)) continue;
      page[e] = p.table[(int64_t)parents[i] * p.stride + c], at[e] = c;
    }
#pragma unroll
    for (int e = 0; e < kForkEach; ++e) {
      if (at[e] < 0) continue;
      const int i = (e * kPlanThreads + (int)threadIdx.x) / max(p.width, 1);
      const bool real = (unsigned)page[e] < (unsigned)p.pages;
      p.table[(int64_t)names[i] * p.stride + at[e]] = real ? page[e] : -1;
      if (real) __hip_atomic_fetch_add(p.refs + page[e], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = e * kPlanThreads + threadIdx.x;
    if (i >= count) continue;
    if (n[e] >= 0) p.lens[names[i]] = n[e];
    if (done) done[i] = n[e] >= 0;
  }
}

// ---------------------------------------------------------------- extend ---

// Scratch: how many pages to copy, from where to where, then the pages handed out.
struct Copies {
  int32_t count, rest[15];
  int32_t src[kMaxRows], dst[kMaxRows];
};

// Page numbers from `at` on: what is at refs[at] .. refs[at + 15], 1 past the pool.
struct Held {
  u32x4 w[4];
  __device__ __forceinline__ void load(const Pages& p, int64_t at) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (at + 4 * i + 4 <= p.pages) {
        w[i] = *reinterpret_cast<const u32x4*>(p.refs + at + 4 * i);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = at + 4 * i + j < p.pages ? (uint32_t)p.refs[at + 4 * i + j] : 1u;
      }
    }
  }
  __device__ __forceinline__ bool is(int i) const { return (int)w[i / 4][i % 4] > 0; }
};
constexpr int kLook = 16 * kPlanThreads;  // pages looked at together

constexpr int kFresh = kClaims;  // new pages that stay in LDS, where the claims were

__global__ __launch_bounds__(kPlanThreads) void extend_kernel(Pages p, const int32_t* rows, const int32_t* add, int32_t* status, int count, int layers,
                                                             Copies* copies, int32_t* many) {
  __shared__ int32_t names[kMaxRows], shared_page[kMaxRows], before[kMaxRows + 1], claims[kClaims];
  __shared__ int lds[kPlanWaves];
  const int each = (count + kPlanThreads - 1) / kPlanThreads;  // consecutive rows of a thread
  const int i0 = threadIdx.x * each;
  int need[kEach], tail[kEach], name[kEach], more[kEach], holders[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = i0 + e;
    need[e] = 0, tail[e] = -1, name[e] = -1, more[e] = 0, holders[e] = 0;
    if (e < each && i < count) name[e] = rows[i], more[e] = max(add[i], 0);
  }
  Held held;
  held.load(p, (int64_t)threadIdx.x * 16);
  const bool few = p.rows <= kClaims;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (e >= each || i0 + e >= count) continue;
    names[i0 + e] = name[e], shared_page[i0 + e] = -1;
    if (few && (unsigned)name[e] < (unsigned)p.rows) claims[name[e]] = 0x7fffffff;
  }
  __syncthreads();
  if (few) {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (e < each && i0 + e < count && (unsigned)name[e] < (unsigned)p.rows) atomicMin(&claims[name[e]], i0 + e);
    __syncthreads();
  }
  bool too_long = false, any_shared = false;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = i0 + e, row = name[e];
    if (e >= each || i >= count || (unsigned)row >= (unsigned)p.rows || more[e] == 0) continue;
    bool again = false;
    if (few) again = claims[row] != i;
    else
      for (int j = 0; j < i; ++j) again |= names[j] == row;
    if (again) continue;
    const int len = max(p.lens[row], 0);
    const int64_t now = (int64_t)len + more[e];
    if (now > capacity(p)) {
      too_long = true;
      continue;
    }
    need[e] = pages_of((int)now, p) - pages_of(len, p);
    tail[e] = len;
    if (len & ((1 << p.shift) - 1)) {
      const int page = p.table[(int64_t)row * p.stride + (len >> p.shift)];
      if ((unsigned)page < (unsigned)p.pages) holders[e] = p.refs[page];
      if (holders[e] > 1) shared_page[i] = page, any_shared = true;
    }
  }
  too_long = __syncthreads_or(too_long);
  any_shared = __syncthreads_or(any_shared);
  int copied = 0;  // bit e
  if (any_shared) {
    // all but the last of a page's holders take a copy (1024 rows that share one page 42 us, 4096 326)
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = i0 + e;
      if (e >= each || i >= count || shared_page[i] < 0) continue;
      int rank = 0;
      for (int j = 0; j < i; ++j) rank += shared_page[j] == shared_page[i];
      if (rank < holders[e] - 1) copied |= 1 << e;
    }
  }
  int sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    need[e] += copied >> e & 1;
    sum += need[e];
  }
  int total, all_copies = 0;
  int at = block_scan(sum, lds, total), copy_at = 0;
  if (any_shared) copy_at = block_scan(__builtin_popcount(copied), lds, all_copies);
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (e < each && i0 + e < count) {
      before[i0 + e] = at | (copied >> e & 1) << 31;
      at += need[e];
    }
  // the lowest free pages; the claims are read no more
  int32_t* fresh = total <= kFresh ? claims : many;
  int found = 0;
  for (int64_t base = 0; found < total && base < p.pages; base += kLook) {
    const Held now = held;
    held.load(p, base + kLook + (int64_t)threadIdx.x * 16);
    int n = 0, all;
#pragma unroll
    for (int j = 0; j < 16; ++j) n += !now.is(j);
    int rank = found + block_scan(n, lds, all);
    found += all;
    if (rank < total) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (!now.is(j)) {
          if (rank < total) fresh[rank] = (int32_t)(base + threadIdx.x * 16 + j);
          ++rank;
        }
    }
  }
  const int say = too_long ? -1 : all_copies && !layers ? -2 : max(total - found, 0);
  if (threadIdx.x == 0) *status = say, copies->count = say ? 0 : all_copies;
  if (say) return;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = i0 + e;
    if (e >= each || i >= count || tail[e] < 0) continue;
    if (copied >> e & 1) {
      const int to = fresh[before[i] & 0x7fffffff], from = shared_page[i];
      copies->src[copy_at] = from, copies->dst[copy_at] = to;
      ++copy_at;
      p.table[(int64_t)name[e] * p.stride + (tail[e] >> p.shift)] = to;
      p.refs[to] = 1;
      __hip_atomic_fetch_add(p.refs + from, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    shared_page[i] = pages_of(tail[e], p) - (copied >> e & 1);  // the column of its first page
    p.lens[name[e]] = tail[e] + more[e];
  }
  __syncthreads();
  for (int k = threadIdx.x; k < total; k += kPlanThreads) {
    int lo = 0, hi = count;  // the row that page k goes to: the last that begins at or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if ((before[mid] & 0x7fffffff) <= k) lo = mid; else hi = mid;
    }
    const int at = k - (before[lo] & 0x7fffffff);
    if (before[lo] < 0 && at == 0) continue;  // the copy
    const int page = fresh[k];
    p.table[(int64_t)names[lo] * p.stride + shared_page[lo] + at] = page;
    p.refs[page] = 1;
  }
}

// --------------------------------------------------------------- compact ---

// The pages in use behind the first `used` move to the free places among them,
// lowest to lowest; place[page] is the rank of a page that moves, -1 of others.
__global__ __launch_bounds__(kPlanThreads) void compact_kernel(Pages p, int32_t* used_out, int32_t* count, int32_t* src, int32_t* dst, int32_t* place) {
  __shared__ int lds[kPlanWaves];
  int n = 0, used;
  for (int64_t at = (int64_t)threadIdx.x * 16; at < p.pages; at += kLook) {
    Held h;
    h.load(p, at);
#pragma unroll
    for (int j = 0; j < 16; ++j) n += at + j < p.pages && h.is(j);
  }
  block_scan(n, lds, used);
  int moved = 0, gaps = 0;
  for (int64_t base = 0; base < p.pages; base += kLook) {
    const int64_t at = base + threadIdx.x * 16;
    Held h;
    h.load(p, at);
    int free = 0, go = 0, all;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      free += at + j < used && !h.is(j);
      go += at + j >= used && at + j < p.pages && h.is(j);
    }
    const int ranks = block_scan(free | go << 16, lds, all);  // at most 2^14 each
    int to = gaps + (ranks & 0xffff), from = moved + (ranks >> 16);
    gaps += all & 0xffff, moved += all >> 16;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (at + j >= p.pages) break;
      const bool goes = at + j >= used && h.is(j);
      place[at + j] = goes ? from : -1;
      if (goes) src[from++] = (int32_t)(at + j);
      if (at + j < used && !h.is(j)) dst[to++] = (int32_t)(at + j);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moved; i += kPlanThreads) {
    p.refs[dst[i]] = p.refs[src[i]];
    p.refs[src[i]] = 0;
  }
  if (threadIdx.x == 0) *count = moved, *used_out = used;
}

// ---------------------------------------------------------------- copies ---

constexpr int kLaunchLayers = 32;
struct Layers {
  lb_kv8_layer at[kLaunchLayers];
};
constexpr int kPieceBytes = 16384;

// Pages src[i] to dst[i] in `layers` layers, sixteen KB a workgroup and turn; the first
// `table_blocks` workgroups put the pages that moved into the tables instead.
__global__ __launch_bounds__(256) void copy_kernel(Pages p, int table_blocks, const int32_t* place, const int32_t* count, int most, const int32_t* src,
                                                   const int32_t* dst, Layers layers, int num_layers, int heads, int page_bytes) {
  if ((int)blockIdx.x < table_blocks) {
    const int64_t all = (int64_t)p.rows * p.width;
    for (int64_t x = blockIdx.x * 256 + threadIdx.x; x < all; x += (int64_t)table_blocks * 256) {
      int32_t* at = p.table + x / p.width * p.stride + x % p.width;
      const int page = *at;
      if ((unsigned)page >= (unsigned)p.pages) continue;
      const int i = place[page];
      if (i >= 0) *at = dst[i];
    }
    return;
  }
  const int pairs = count ? min(*count, most) : most, pieces = (page_bytes + kPieceBytes - 1) / kPieceBytes;
  const int64_t units = (int64_t)pairs * num_layers * 2 * pieces;
  for (int64_t u = blockIdx.x - table_blocks; u < units; u += gridDim.x - table_blocks) {
    const int piece = u % pieces;
    int64_t rest = u / pieces;
    const bool values = rest & 1;
    rest >>= 1;
    const int layer = rest % num_layers, pair = rest / num_layers;
    const int from = src[pair], to = dst[pair];
    if ((unsigned)from >= (unsigned)p.pages || (unsigned)to >= (unsigned)p.pages || from == to) continue;
    int8_t* cache = values ? layers.at[layer].v_cache : layers.at[layer].k_cache;
    float* scale = values ? layers.at[layer].v_scale : layers.at[layer].k_scale;
    const u32x4* x = reinterpret_cast<const u32x4*>(cache + (int64_t)from * page_bytes) + piece * (kPieceBytes / 16);
    u32x4* y = reinterpret_cast<u32x4*>(cache + (int64_t)to * page_bytes) + piece * (kPieceBytes / 16);
    const int n = min(kPieceBytes, page_bytes - piece * kPieceBytes) / 16;
    u32x4 w[kPieceBytes / 4096];
#pragma unroll
    for (int j = 0; j < kPieceBytes / 4096; ++j)
      if (j * 256 + (int)threadIdx.x < n) w[j] = x[j * 256 + threadIdx.x];
#pragma unroll
    for (int j = 0; j < kPieceBytes / 4096; ++j)
      if (j * 256 + (int)threadIdx.x < n) y[j * 256 + threadIdx.x] = w[j];
    if (piece == 0)
      for (int h = threadIdx.x; h < heads; h += 256) scale[(int64_t)to * heads + h] = scale[(int64_t)from * heads + h];
  }
}

struct LayerShape {
  const lb_kv8_layer* at;
  int64_t count, heads, page_bytes;
};

int check_layers(const lb_kv8_layer* at, int64_t count, int64_t num_pages, int64_t heads, int64_t page_size, int64_t head_dim) {
  if (count < 0) return LB_ERR_ARG;
  if (count == 0) return LB_OK;
  if (!at || heads <= 0 || heads > 4096) return LB_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LB_ERR_PROB_SHAPE;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return LB_ERR_PROB_SHAPE;
  for (int64_t i = 0; i < count && num_pages > 0; ++i) {
    if (!at[i].k_cache || !at[i].v_cache || !at[i].k_scale || !at[i].v_scale) return LB_ERR_ARG;
    if (!lbh::aligned(at[i].k_cache, 16) || !lbh::aligned(at[i].v_cache, 16) || !lbh::aligned(at[i].k_scale, 4) || !lbh::aligned(at[i].v_scale, 4))
      return LB_ERR_ALIGN;
  }
  return LB_OK;
}

// The copies, thirty-two layers a launch; the tables in the first of them.
void copy(const Pages& p, const LayerShape& s, const int32_t* place, const int32_t* count, int64_t most, const int32_t* src, const int32_t* dst,
          hipStream_t st) {
  const int64_t cus = lbh::device_cus();
  int table_blocks = 0;
  if (place) {
    const int64_t blocks = ((int64_t)p.rows * p.width + 1023) / 1024;
    table_blocks = (int)(blocks < cus ? blocks : cus);
  }
  for (int64_t first = 0; first < s.count || (first == 0 && table_blocks); first += kLaunchLayers) {
    Layers layers = {};
    const int n = (int)(s.count - first < kLaunchLayers ? s.count - first : kLaunchLayers);
    for (int i = 0; i < n; ++i) layers.at[i] = s.at[first + i];
    const int64_t units = most * n * 2 * ((s.page_bytes + kPieceBytes - 1) / kPieceBytes), wide = 8 * cus;
    const int64_t grid = table_blocks + (units < wide ? units : wide);
    if (grid > 0)
      copy_kernel<<<dim3((unsigned)grid), dim3(256), 0, st>>>(p, table_blocks, place, count, (int)most, src, dst, layers, n, (int)s.heads, (int)s.page_bytes);
    table_blocks = 0;
  }
}

int check_pages(const int32_t* table, int64_t rows, int64_t max_pages, int64_t stride, const int32_t* lens, const int32_t* refs, int64_t num_pages,
                int64_t page_size) {
  if (rows < 0 || rows > 0x7fffffff || max_pages < 0 || stride < max_pages || num_pages < 0 || num_pages > 0x7fffffff - 65536) return LB_ERR_ARG;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return LB_ERR_PROB_SHAPE;
  if (max_pages > (1 << 28) / page_size) return LB_ERR_ARG;
  if ((!table && rows * max_pages > 0) || (!lens && rows > 0) || (!refs && num_pages > 0)) return LB_ERR_ARG;
  return lbh::aligned(refs, 16) ? LB_OK : LB_ERR_ALIGN;
}

Pages pages_at(int32_t* table, int64_t rows, int64_t max_pages, int64_t stride, int32_t* lens, int32_t* refs, int64_t num_pages, int64_t page_size) {
  Pages p;
  p.table = table, p.lens = lens, p.refs = refs, p.stride = stride;
  p.rows = (int)rows, p.width = (int)max_pages, p.pages = (int)num_pages;
  p.shift = page_size > 0 ? __builtin_ctzll((unsigned long long)page_size) : 0;
  return p;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace
}  // namespace lb

extern "C" int lb_kv8_pages_free(int32_t* page_table, int64_t rows, int64_t max_pages, int64_t table_stride, int32_t* seq_lens, int32_t* refs,
                                 int64_t num_pages, int64_t page_size, const int32_t* which, const int32_t* keep, int64_t count, lb_stream_t stream) {
  using namespace lb;
  const int err = check_pages(page_table, rows, max_pages, table_stride, seq_lens, refs, num_pages, page_size);
  if (err != LB_OK) return err;
  if (count < 0 || count > kMaxRows || (count > 0 && !which)) return LB_ERR_ARG;
  if (count == 0 || rows == 0) return LB_OK;
  const Pages p = pages_at(page_table, rows, max_pages, table_stride, seq_lens, refs, num_pages, page_size);
  free_kernel<<<dim3((unsigned)count, col_blocks(max_pages)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream)>>>(p, which, keep);
  return lbh::launch_status();
}

extern "C" int lb_kv8_pages_fork(int32_t* page_table, int64_t rows, int64_t max_pages, int64_t table_stride, int32_t* seq_lens, int32_t* refs,
                                 int64_t num_pages, int64_t page_size, const int32_t* parents, const int32_t* children, const int32_t* lens,
                                 int32_t* done, int64_t count, lb_stream_t stream) {
  using namespace lb;
  const int err = check_pages(page_table, rows, max_pages, table_stride, seq_lens, refs, num_pages, page_size);
  if (err != LB_OK) return err;
  if (count < 0 || count > kMaxRows || (count > 0 && (!parents || !children))) return LB_ERR_ARG;
  if (count == 0) return LB_OK;
  const Pages p = pages_at(page_table, rows, max_pages, table_stride, seq_lens, refs, num_pages, page_size);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (count * max_pages <= kForkEntries) {
    fork_lens_kernel<true><<<dim3(1), dim3(kPlanThreads), 0, st>>>(p, parents, children, lens, done, (int)count);
  } else {
    fork_kernel<<<dim3((unsigned)count, col_blocks(max_pages)), dim3(256), 0, st>>>(p, parents, children, lens);
    fork_lens_kernel<false><<<dim3(1), dim3(kPlanThreads), 0, st>>>(p, parents, children, lens, done, (int)count);
  }
  return lbh::launch_status();
}

extern "C" size_t lb_kv8_pages_extend_scratch_bytes(int64_t num_pages) {
  return num_pages < 0 ? 0 : lb::up256(sizeof(lb::Copies)) + lb::up256((size_t)num_pages * 4);
}

extern "C" int lb_kv8_pages_extend(int32_t* page_table, int64_t rows, int64_t max_pages, int64_t table_stride, int32_t* seq_lens, int32_t* refs,
                                   int64_t num_pages, int64_t page_size, const int32_t* which, const int32_t* add, int64_t count, int32_t* status,
                                   const lb_kv8_layer* layers, int64_t num_layers, int64_t heads_kv, int64_t head_dim, void* scratch,
                                   size_t scratch_bytes, lb_stream_t stream) {
  using namespace lb;
  int err = check_pages(page_table, rows, max_pages, table_stride, seq_lens, refs, num_pages, page_size);
  if (err == LB_OK) err = check_layers(layers, num_layers, num_pages, heads_kv, page_size, head_dim);
  if (err != LB_OK) return err;
  if (count < 0 || count > kMaxRows || (count > 0 && (!which || !add)) || !status) return LB_ERR_ARG;
  if (count * max_pages > (1 << 30)) return LB_ERR_PROB_SHAPE;  // new pages are numbered in 32 bits
  if (!lbh::aligned(scratch, 16)) return LB_ERR_ALIGN;
  if (!scratch || scratch_bytes < lb_kv8_pages_extend_scratch_bytes(num_pages)) return LB_ERR_SCRATCH;
  const Pages p = pages_at(page_table, rows, max_pages, table_stride, seq_lens, refs, num_pages, page_size);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  Copies* copies = static_cast<Copies*>(scratch);
  int32_t* fresh = reinterpret_cast<int32_t*>(static_cast<char*>(scratch) + up256(sizeof(Copies)));
  extend_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(p, which, add, status, (int)count, num_layers > 0, copies, fresh);
  copy(p, {layers, num_layers, heads_kv, heads_kv * page_size * head_dim}, nullptr, &copies->count, count, copies->src, copies->dst, st);
  return lbh::launch_status();
}

extern "C" size_t lb_kv8_pages_compact_scratch_bytes(int64_t num_pages) { return num_pages < 0 ? 0 : 256 + 3 * lb::up256((size_t)num_pages * 4); }

extern "C" int lb_kv8_pages_compact(int32_t* page_table, int64_t rows, int64_t max_pages, int64_t table_stride, int32_t* refs, int64_t num_pages,
                                    int32_t* used, const lb_kv8_layer* layers, int64_t num_layers, int64_t heads_kv, int64_t page_size,
                                    int64_t head_dim, void* scratch, size_t scratch_bytes, lb_stream_t stream) {
  using namespace lb;
  int err = check_pages(page_table, rows, max_pages, table_stride, used, refs, num_pages, page_size);  // no lengths here
  if (err == LB_OK) err = check_layers(layers, num_layers, num_pages, heads_kv, page_size, head_dim);
  if (err != LB_OK) return err;
  if (!used) return LB_ERR_ARG;
  if (!lbh::aligned(scratch, 16)) return LB_ERR_ALIGN;
  if (!scratch || scratch_bytes < lb_kv8_pages_compact_scratch_bytes(num_pages)) return LB_ERR_SCRATCH;
  const Pages p = pages_at(page_table, rows, max_pages, table_stride, nullptr, refs, num_pages, page_size);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  int32_t* count = static_cast<int32_t*>(scratch);
  int32_t* src = count + 64;
  int32_t* dst = src + up256((size_t)num_pages * 4) / 4;
  int32_t* place = dst + up256((size_t)num_pages * 4) / 4;
  compact_kernel<<<dim3(1), dim3(kPlanThreads), 0, st>>>(p, used, count, src, dst, place);
  copy(p, {layers, num_layers, heads_kv, heads_kv * page_size * head_dim}, place, count, num_pages / 2, src, dst, st);
  return lbh::launch_status();
}

extern "C" int lb_kv8_copy_pages(const lb_kv8_layer* layers, int64_t num_layers, int64_t num_pages, int64_t heads_kv, int64_t page_size, int64_t head_dim,
                                 const int32_t* src, const int32_t* dst, int64_t count, lb_stream_t stream) {
  using namespace lb;
  const int err = check_layers(layers, num_layers, num_pages, heads_kv, page_size, head_dim);
  if (err != LB_OK) return err;
  if (num_pages < 0 || num_pages > 0x7fffffff - 65536 || count < 0 || count > 0x7fffffff || (count > 0 && (!src || !dst))) return LB_ERR_ARG;
  if (count == 0 || num_layers == 0 || num_pages == 0) return LB_OK;
  const Pages p = pages_at(nullptr, 0, 0, 0, nullptr, nullptr, num_pages, page_size);
  copy(p, {layers, num_layers, heads_kv, heads_kv * page_size * head_dim}, nullptr, nullptr, count, src, dst, reinterpret_cast<hipStream_t>(stream));
  return lbh::launch_status();
}
