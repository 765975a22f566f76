// Writer of the paged 8-bit cache: rotates queries and keys to their positions
// and stores keys and values as codes, one launch for both.
//
//   q'  = R(pos) q,  k' = R(pos) k    R(pos): pairs (a, b) of the first rot values of a
//                                     head become (a cos - b sin, b cos + a sin)
//   s   = max(s_old if the page holds earlier tokens, max |x| / 127)   per page, head; K and V apart
//   old = rint(old * s_old / s) where s grew
//   c   = rint(x / s)
//
// The rotation and the codes are computed with each product and sum rounded to
// fp32 by itself (no contraction), so a program that repeats the definition in
// 32 bits gets the same codes.
//
// Bound by memory: each row is read and written once.  A workgroup holds one head
// of one page, keys or values, in registers, since every code waits for the
// page's largest value; the workgroups of the queries run beside them.  16384
// tokens, 40 / 8 heads of 128: 102 us, 4.5 TB/s where a large copy reaches 5.0; one
// token: 5.2 us, a launch and the loads that wait for one another (length, page,
// scale and rows).
#include "attn_common.hpp"

namespace lb {
namespace {

struct Rows {  // fp16 [tokens][heads][head_dim], the last axis contiguous
  uint16_t* p;
  int64_t token, head;  // strides in elements
};

struct AppendArgs {
  Rows q, k, v, q_out, k_out;
  int8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  const int32_t *page_table, *seq_lens, *starts;
  const float* cos_sin;
  int64_t table_stride;
  int num_pages, page_shift, max_pages;
  int batch, tokens, heads_q, heads_kv, d8;  // d8: head_dim / 8
  int positions, rot, interleaved;
  int per_seq;    // tokens of each sequence where starts is null
  int kv_blocks;  // workgroups of the keys and values, before those of the queries
  int page_bound;  // pages a sequence can touch (starts null)
  int q_heads_per_thread;
};

typedef float f32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x8 load8(const uint16_t* p) {
  const u32x4 w = *reinterpret_cast<const u32x4*>(p);
  f32x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 h = as_h2(w[i]);
    r[2 * i] = (float)h[0];
    r[2 * i + 1] = (float)h[1];
  }
  return r;
}

__device__ __forceinline__ void store8(uint16_t* p, f32x8 v) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = as_u32((f16x2){(f16)v[2 * i], (f16)v[2 * i + 1]});
  *reinterpret_cast<u32x4*>(p) = w;
}

// (x, y) -> (x cos - y sin, y cos + x sin), every operation rounded by itself.
__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
#pragma clang fp contract(off)
  const float xc = x * c, ys = y * s, yc = y * c, xs = x * s;
  x = xc - ys;
  y = yc + xs;
}

// Two vectors of eight of a head and their angles.  Halves pair value i with
// i + rot/2: vectors (j, j + rot/16), with eight angles.  Interleaved pairs are
// neighbours inside a vector: (j, j + head_dim/16), with four angles each.  Either
// way, and past the rotated part, neighbouring j take neighbouring vectors, so
// that loads and stores cover whole lines.
struct Pair {
  int v0, v1;
  bool r0, r1;  // rotated
};
__device__ __forceinline__ Pair pair_of(const AppendArgs& a, int j) {
  const int n = a.rot / 16, half = a.d8 / 2;
  if (a.interleaved) return {j, j + half, j < 2 * n, j + half < 2 * n};
  if (j < n) return {j, j + n, true, true};
  return {n + j, half + j, false, false};
}

// The pair's cos and sin at `pos` (interleaved: four of v0, then four of v1).  A
// position outside the table has none: NaN, which the outputs then show.
__device__ __forceinline__ void angles(const AppendArgs& a, int pos, const Pair& p, f32x8& c, f32x8& s) {
  if ((unsigned)pos >= (unsigned)a.positions) {
    c = s = (f32x8)(__builtin_nanf(""));
    return;
  }
  const float* row = a.cos_sin + (int64_t)pos * a.rot;
  const int f0 = a.interleaved ? 4 * p.v0 : 8 * p.v0, f1 = a.interleaved ? (p.r1 ? 4 * p.v1 : f0) : f0 + 4;
  const f32x4 c0 = *reinterpret_cast<const f32x4*>(row + f0), c1 = *reinterpret_cast<const f32x4*>(row + f1);
  const f32x4 s0 = *reinterpret_cast<const f32x4*>(row + a.rot / 2 + f0);
  const f32x4 s1 = *reinterpret_cast<const f32x4*>(row + a.rot / 2 + f1);
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = c0[i], c[4 + i] = c1[i], s[i] = s0[i], s[4 + i] = s1[i];
}

__device__ __forceinline__ void rotate_pair(const Pair& p, bool interleaved, f32x8& x, f32x8& y, const f32x8& c,
                                            const f32x8& s) {
  if (!p.r0) return;
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float u = x[2 * i], w = x[2 * i + 1];
      turn(u, w, c[i], s[i]);
      x[2 * i] = u, x[2 * i + 1] = w;
    }
    if (!p.r1) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float u = y[2 * i], w = y[2 * i + 1];
      turn(u, w, c[4 + i], s[4 + i]);
      y[2 * i] = u, y[2 * i + 1] = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float u = x[i], w = y[i];
      turn(u, w, c[i], s[i]);
      x[i] = u, y[i] = w;
    }
  }
}

__device__ __forceinline__ int code_of(float x, float inverse) {
  const float r = __builtin_rintf(x * inverse);
  return (int)__builtin_fminf(__builtin_fmaxf(r, -127.0f), 127.0f);
}

__device__ __forceinline__ int byte_of(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }

// Largest bit pattern of |x| over the workgroup: above the infinity's pattern
// if any is NaN, so a non-finite value shows in the page's scale.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* lds) {
  const int lane = lane_id();
#pragma unroll
  for (int x = 1; x < kWave; x *= 2) {
    const uint32_t o = from_lane(v, lane ^ x);
    v = o > v ? o : v;
  }
  const int waves = blockDim.x / kWave;
  if (waves == 1) return v;
  if (lane == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int i = 0; i < waves; ++i) v = lds[i] > v ? lds[i] : v;
  return v;
}

// One head of one page: where it is, which of its slots are new, and the scale
// that it has and gets.
struct Cell {
  int page_lo, lo, hi;  // positions: of the page's first slot, and of the new tokens in it
  int start, first;     // of the sequence's new tokens: the first's position, and its row
  int head;
  bool stored;          // the page is one of the cache; else its tokens' keys are only returned
  int64_t cell;         // page * heads + head
  float* scale_at;
  float old_scale;
  bool kept;            // the page holds earlier tokens
  __device__ __forceinline__ bool is_new(int pos) const { return pos >= lo && pos < hi; }
  __device__ __forceinline__ int old_slots() const { return kept ? start - page_lo : 0; }
};

// What the page's codes are scaled by.  `peak` is the largest bit pattern of a
// new value; every thread of the workgroup calls this.
struct Scaling {
  float inverse, shrink;
  bool grew;
};
__device__ __forceinline__ Scaling rescale(const Cell& c, uint32_t peak, uint32_t* lds) {
  peak = block_max(peak, lds);
  const float need = __builtin_bit_cast(float, peak) * (1.0f / 127.0f);
  // NaN on either side stays: a page that held it once has no codes to rescale
  const float scale = need <= c.old_scale || c.old_scale != c.old_scale ? c.old_scale : need;
  Scaling s;
  s.grew = c.kept && scale != c.old_scale && c.old_scale == c.old_scale;
  if (threadIdx.x == 0 && (scale != c.old_scale || !c.kept)) *c.scale_at = scale;
  s.inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
  s.shrink = s.grew ? c.old_scale / scale : 1.0f;
  return s;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// Rows of k_out are the page's workgroup's too, which holds the rotated keys:
// also those of a page that is absent, or past the table, and the zeros of padding
// (pages before position 0).
//
// Keys: a thread holds two neighbouring tokens at a pair of vectors that rotate
// together, so each value and angle is loaded once; eight codes of a token are
// one store of the layout [page][token][channel].
__device__ __forceinline__ void append_keys(const AppendArgs& a, const Cell& c, uint32_t* lds) {
  const int pairs = a.d8 / 2;
  const int tid = threadIdx.x;
  const int j = tid % pairs, off0 = 2 * (tid / pairs);
  const bool active = off0 < 1 << a.page_shift;
  const Pair pr = pair_of(a, j);
  f32x8 x[2][2];
  uint32_t peak = 0;
  if (active && c.page_lo + off0 + 2 > c.lo && c.page_lo + off0 < c.hi) {
    f32x8 cs[2], sn[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // a slot that is not new reads the row of one that is, and drops it
      const int pos = min(max(c.page_lo + off0 + i, c.lo), c.hi - 1);
      const uint16_t* row = a.k.p + (int64_t)(c.first + (pos - c.start)) * a.k.token + (int64_t)c.head * a.k.head;
      x[i][0] = load8(row + 8 * pr.v0), x[i][1] = load8(row + 8 * pr.v1);
      if (pr.r0) angles(a, pos, pr, cs[i], sn[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      rotate_pair(pr, a.interleaved, x[i][0], x[i][1], cs[i], sn[i]);
      const int pos = c.page_lo + off0 + i;
      if (!c.is_new(pos)) continue;
      if (a.k_out.p) {
        if (c.page_lo < 0) x[i][0] = x[i][1] = (f32x8)(0.0f);
        uint16_t* out = a.k_out.p + (int64_t)(c.first + (pos - c.start)) * a.k_out.token + (int64_t)c.head * a.k_out.head;
        store8(out + 8 * pr.v0, x[i][0]);
        store8(out + 8 * pr.v1, x[i][1]);
      }
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t m = magnitude(x[i][v][e]);
          peak = m > peak ? m : peak;
        }
    }
  }
  if (!c.stored) return;
  const Scaling s = rescale(c, peak, lds);
  if (!active) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      u32x2* at = reinterpret_cast<u32x2*>(a.k_cache + ((c.cell << a.page_shift) + off0 + i) * (8 * a.d8) +
                                           8 * (v ? pr.v1 : pr.v0));
      u32x2 w = {0, 0};
      if (c.is_new(c.page_lo + off0 + i)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e / 4] |= (uint32_t)(code_of(x[i][v][e], s.inverse) & 255) << (8 * (e % 4));
        *at = w;
      } else if (s.grew && off0 + i < c.old_slots()) {
        const u32x2 old = *at;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[e / 4] |= (uint32_t)(code_of((float)byte_of(old[e / 4], e % 4), s.shrink) & 255) << (8 * (e % 4));
        *at = w;
      }
    }
}

// Values: a thread holds four neighbouring tokens at eight neighbouring
// channels; four codes of a channel are one store of the layout
// [page][channel][token].
__device__ __forceinline__ void append_values(const AppendArgs& a, const Cell& c, uint32_t* lds) {
  const int t4 = (1 << a.page_shift) / 4;
  const int tid = threadIdx.x;
  const int d8 = tid / t4, off0 = 4 * (tid % t4);
  const bool active = d8 < a.d8;
  const int pos0 = c.page_lo + off0;
  const bool any_new = active && pos0 + 4 > c.lo && pos0 < c.hi;
  f32x8 x[4];
  uint32_t peak = 0;
  if (any_new) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = min(max(pos0 + i, c.lo), c.hi - 1);
      x[i] = load8(a.v.p + (int64_t)(c.first + (pos - c.start)) * a.v.token + (int64_t)c.head * a.v.head + 8 * d8);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c.is_new(pos0 + i))
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t m = magnitude(x[i][e]);
          peak = m > peak ? m : peak;
        }
  }
  const Scaling s = rescale(c, peak, lds);
  const bool olds = active && s.grew && off0 < c.old_slots();
  if (!any_new && !olds) return;
  int8_t* base = a.v_cache + ((c.cell * (8 * a.d8) + 8 * d8) << a.page_shift) + off0;
  const bool full = c.is_new(pos0) && c.is_new(pos0 + 3);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    int8_t* at = base + ((int64_t)e << a.page_shift);
    uint32_t w = 0;
    if (full) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= (uint32_t)(code_of(x[i][e], s.inverse) & 255) << (8 * i);
      *reinterpret_cast<uint32_t*>(at) = w;
    } else if (olds) {
      const uint32_t old = *reinterpret_cast<const uint32_t*>(at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int code = byte_of(old, i);
        if (c.is_new(pos0 + i)) code = code_of(x[i][e], s.inverse);
        else if (off0 + i < c.old_slots()) code = code_of((float)code, s.shrink);
        w |= (uint32_t)(code & 255) << (8 * i);
      }
      *reinterpret_cast<uint32_t*>(at) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c.is_new(pos0 + i)) at[i] = (int8_t)code_of(x[i][e], s.inverse);
    }
  }
}

// The first of sequence b's packed tokens.
__device__ __forceinline__ int first_of(const AppendArgs& a, int b) { return max(a.starts[b], 0); }

// Rows of padding (a token before position 0) come out as zeros.
__device__ __forceinline__ void rotate_queries(const AppendArgs& a, int64_t job) {
  const int pairs = a.d8 / 2;
  const int j = (int)(job % pairs);
  const int64_t rest = job / pairs;
  const int chunks = (a.heads_q + a.q_heads_per_thread - 1) / a.q_heads_per_thread;
  const int chunk = (int)(rest % chunks);
  const int64_t t64 = rest / chunks;
  if (t64 >= a.tokens) return;
  const int t = (int)t64;
  int b, first, n;
  if (a.starts == nullptr) {
    b = t / a.per_seq, first = b * a.per_seq, n = a.per_seq;
  } else {
    int lo = 0, hi = a.batch;  // the last b in [0, batch] with starts[b] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.starts[mid] <= t) lo = mid; else hi = mid;
    }
    b = lo, first = first_of(a, b), n = a.starts[b + 1] - first;
    if (t < first || t >= first + n) return;  // outside every sequence
  }
  const int pos = max(a.seq_lens[b], 0) - n + (t - first);
  const Pair pr = pair_of(a, j);
  f32x8 c, s;
  if (pr.r0) angles(a, pos, pr, c, s);
  const int h0 = chunk * a.q_heads_per_thread, h1 = min(h0 + a.q_heads_per_thread, a.heads_q);
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const uint16_t* row = a.q.p + (int64_t)t * a.q.token + (int64_t)h * a.q.head;
    uint16_t* out = a.q_out.p + (int64_t)t * a.q_out.token + (int64_t)h * a.q_out.head;
    f32x8 x = load8(row + 8 * pr.v0), y = load8(row + 8 * pr.v1);
    rotate_pair(pr, a.interleaved, x, y, c, s);
    if (pos < 0) x = y = (f32x8)(0.0f);
    store8(out + 8 * pr.v0, x);
    store8(out + 8 * pr.v1, y);
  }
}

// The packed sequence that holds item `item` of the pages, where sequence b's
// begin at item starts[b] / page_size + 2 b (rising for sorted starts): the last b
// that begins at or before it, -1 if none does.  The whole wave searches together,
// 64 sequences a load; `item` is wave-uniform.
__device__ __forceinline__ int sequence_of_item(const AppendArgs& a, int item) {
  const int lane = lane_id();
  int count = 0;
  for (int c = 0; c < a.batch; c += kWave) {
    const int b = c + lane;
    const bool le = b < a.batch && first_of(a, b) / (1 << a.page_shift) + 2 * b <= item;
    const uint64_t m = __ballot(le);
    count += __popcll(m);
    if (m != ~0ull) break;
  }
  return __builtin_amdgcn_readfirstlane(count) - 1;
}

__global__ __launch_bounds__(1024) void kv8_append_kernel(AppendArgs a) {
  __shared__ uint32_t lds[16];
  if ((int)blockIdx.x >= a.kv_blocks) {
    rotate_queries(a, (int64_t)(blockIdx.x - a.kv_blocks) * blockDim.x + threadIdx.x);
    return;
  }
  // workgroup -> (page item, head, keys or values)
  const int kind = blockIdx.x & 1;
  const int rest = blockIdx.x >> 1;
  const int head = rest % a.heads_kv, item = rest / a.heads_kv;
  int b, first, n, page;
  if (a.starts == nullptr) {
    b = item / a.page_bound, page = item % a.page_bound;
    first = b * a.per_seq, n = a.per_seq;
  } else {
    b = sequence_of_item(a, item);
    if (b < 0) return;
    // the last of the n may not be given: those that are keep their places
    first = first_of(a, b), n = a.starts[b + 1] - first;
    page = item - (first / (1 << a.page_shift) + 2 * b);
    if (n <= 0) return;
  }
  const int len = max(a.seq_lens[b], 0);
  const int start = len - n;  // before position 0 where the first tokens are padding
  page += start >> a.page_shift;
  Cell c;
  c.page_lo = page * (1 << a.page_shift);
  c.lo = max(start, c.page_lo), c.hi = min(min(len, start + (a.tokens - first)), c.page_lo + (1 << a.page_shift));
  if (c.lo >= c.hi) return;
  int id = -1;
  if ((unsigned)page < (unsigned)a.max_pages) id = a.page_table[(int64_t)b * a.table_stride + page];
  c.stored = (unsigned)id < (unsigned)a.num_pages;
  if (!c.stored && (kind == 1 || a.k_out.p == nullptr)) return;
  c.start = start, c.first = first, c.head = head;
  c.cell = (int64_t)id * a.heads_kv + head;
  c.scale_at = (kind == 0 ? a.k_scale : a.v_scale) + c.cell;
  c.kept = c.stored && c.page_lo < start;
  c.old_scale = c.kept ? *c.scale_at : 0.0f;
  if (kind == 0) append_keys(a, c, lds);
  else append_values(a, c, lds);
}

}  // namespace
}  // namespace lb

extern "C" int lb_kv8_append(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, const uint16_t* k,
                             int64_t k_token_stride, int64_t k_head_stride, const uint16_t* v, int64_t v_token_stride,
                             int64_t v_head_stride, uint16_t* q_out, int64_t qo_token_stride, int64_t qo_head_stride,
                             uint16_t* k_out, int64_t ko_token_stride, int64_t ko_head_stride, int8_t* k_cache,
                             int8_t* v_cache, float* k_scale, float* v_scale, int64_t num_pages, int64_t page_size,
                             const int32_t* page_table, int64_t max_pages, int64_t table_stride,
                             const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t batch, int64_t tokens,
                             int64_t heads_q, int64_t heads_kv, int64_t head_dim, const float* cos_sin,
                             int64_t positions, int64_t rot_dim, int32_t interleaved, lb_stream_t stream) {
  using namespace lb;
  constexpr int64_t kIntMax = 0x7fffffff;
  if (batch < 0 || tokens < 0 || heads_q < 0 || heads_kv <= 0 || num_pages < 0 || max_pages < 0 || rot_dim < 0 ||
      positions < 0)
    return LB_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LB_ERR_PROB_SHAPE;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return LB_ERR_PROB_SHAPE;
  if (rot_dim > head_dim || rot_dim % 16 != 0) return LB_ERR_PROB_SHAPE;
  if (heads_q > 4096 || heads_kv > 4096 || batch > (1 << 20) || tokens > (1 << 26) || num_pages > kIntMax ||
      max_pages > kIntMax / page_size || positions > kIntMax || table_stride < max_pages)
    return LB_ERR_ARG;
  if (tokens == 0 || batch == 0) return LB_OK;
  if (cu_seqlens == nullptr && tokens % batch != 0) return LB_ERR_ARG;
  const bool queries = q_out != nullptr && heads_q > 0;
  if (!k || !v || !seq_lens || (queries && !q) || (rot_dim > 0 && !cos_sin)) return LB_ERR_ARG;
  // a cache or a table of nothing has no address: no token has a page then
  if (max_pages > 0 && !page_table) return LB_ERR_ARG;
  if (max_pages > 0 && num_pages > 0 && (!k_cache || !v_cache || !k_scale || !v_scale)) return LB_ERR_ARG;
  // a slot that is not new reads a neighbour's row (and drops it), which that one's thread would be writing
  if (k_out == k) return LB_ERR_ARG;
  const void* ptrs[] = {k, v, queries ? q : nullptr, q_out, k_out, k_cache, v_cache, cos_sin};
  for (const void* p : ptrs)
    if (!lbh::aligned(p, 16)) return LB_ERR_ALIGN;
  int64_t strides = k_token_stride | k_head_stride | v_token_stride | v_head_stride;
  if (queries) strides |= q_token_stride | q_head_stride | qo_token_stride | qo_head_stride;
  if (k_out) strides |= ko_token_stride | ko_head_stride;
  if (strides % 8 != 0) return LB_ERR_ALIGN;

  AppendArgs a;
  a.q = {const_cast<uint16_t*>(q), q_token_stride, q_head_stride};
  a.k = {const_cast<uint16_t*>(k), k_token_stride, k_head_stride};
  a.v = {const_cast<uint16_t*>(v), v_token_stride, v_head_stride};
  a.q_out = {q_out, qo_token_stride, qo_head_stride};
  a.k_out = {k_out, ko_token_stride, ko_head_stride};
  a.k_cache = k_cache, a.v_cache = v_cache, a.k_scale = k_scale, a.v_scale = v_scale;
  a.page_table = page_table, a.seq_lens = seq_lens, a.starts = cu_seqlens, a.cos_sin = cos_sin;
  a.table_stride = table_stride, a.num_pages = (int)num_pages, a.max_pages = (int)max_pages;
  a.page_shift = __builtin_ctzll((unsigned long long)page_size);
  a.batch = (int)batch, a.tokens = (int)tokens, a.heads_q = (int)heads_q, a.heads_kv = (int)heads_kv;
  a.d8 = (int)head_dim / 8, a.positions = (int)positions, a.rot = (int)rot_dim, a.interleaved = interleaved != 0;
  a.per_seq = cu_seqlens ? 0 : (int)(tokens / batch);
  // pages that n tokens can touch: floor((n - 2) / P) + 2 for n >= 1
  a.page_bound = cu_seqlens ? 0 : (int)((a.per_seq - 2 + page_size) / page_size + 1);
  // packed: sequence b's pages are numbered from cu_seqlens[b] / P + 2 b, which leaves room for all of them
  const int64_t items = cu_seqlens ? tokens / page_size + 2 * batch : batch * a.page_bound;
  const int64_t kv_blocks = items * heads_kv * 2;
  const int threads = (int)(page_size * head_dim / 32 < kWave ? kWave : page_size * head_dim / 32);
  // a thread's angles serve several heads once there are threads enough for the
  // chip (16384 tokens, 40 heads: 102 us with eight, 104 with one; 64 tokens: 4.7 us
  // with one, 6.1 with eight)
  const int64_t lanes = tokens * (head_dim / 16);
  const int64_t shared = lanes * heads_q / ((int64_t)lbh::device_cus() * 1024);
  a.q_heads_per_thread = shared < 1 ? 1 : shared > 8 ? 8 : (int)shared;
  const int64_t chunks = (heads_q + a.q_heads_per_thread - 1) / a.q_heads_per_thread;
  const int64_t q_blocks = queries ? (lanes * chunks + threads - 1) / threads : 0;
  if (kv_blocks + q_blocks > kIntMax) return LB_ERR_ARG;
  a.kv_blocks = (int)kv_blocks;
  kv8_append_kernel<<<dim3((unsigned)(kv_blocks + q_blocks)), dim3(threads), 0,
                      reinterpret_cast<hipStream_t>(stream)>>>(a);
  return lbh::launch_status();
}
