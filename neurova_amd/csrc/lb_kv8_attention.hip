// Attention of a sequence's newest tokens over its pages of the 8-bit cache.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= len - n + i
//   k[j] = k_scale[page] ck[j],  v[j] = v_scale[page] cv[j]
//
// The cache is read once, so the bound is its bytes: 2 head_dim a token and
// key/value head.  The query heads of a group and the n tokens are the columns
// of both products, 16 or 32 at a time:
//
//   S^T = K Q^T   rows = tokens: the key layout [token][channel] gives a lane
//                 16 channels of one token in a 16-byte load
//   O^T = V^T P^T rows = channels: the value layout [channel][token] gives a
//                 lane 16 tokens of one channel in a 16-byte load
//
// A wave takes 64 tokens a step.  Token 16 g + 4 t + i is row 4 g + i of
// product t, so the accumulators of lane group g are the tokens 16 g .. 16 g + 15
// of its column, in order: exactly the tokens of the lane's value loads.  The
// weights go from the first product to the second without leaving the lane, and
// a lane's tokens share a page (pages hold 16 tokens or more), so both scales
// are one number a lane and step.
#include "attn_common.hpp"

namespace lb {
namespace {

struct AttnArgs {
  const uint16_t* q;
  int64_t q_token, q_head;
  const int8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int32_t *page_table, *seq_lens;
  uint16_t* out;
  int64_t o_token, o_head;
  int32_t* counters;
  float* parts;
  int64_t table_stride;
  int num_pages, page_shift, max_tokens;
  int batch, new_tokens, heads_kv, group;
  int col_blocks;
  float scale;  // softmax scale * log2(e)
};

constexpr int kStep = 64;           // tokens a wave takes at a time
constexpr int kWaves = 4;
constexpr int kUnit = kStep * kWaves;  // tokens of a unit of work
constexpr float kNoMax = -1e30f;
// The running maximum moves only when a score exceeds it by 2^kSlack, and the
// weights carry 2^kLift more: at most 2^15, inside fp16, and 2^7 farther from its
// subnormals.
constexpr float kSlack = 8.0f;
constexpr int kLift = 7;

// Sixteen signed bytes -> two MFMA fragments of eight fp16 (exact): the byte
// with its sign flipped under the exponent of 1024 is 1024 + 128 + c.
__device__ __forceinline__ void codes_to_half(u32x4 w, f16x8& a, f16x8& b) {
  u32x4 lo, hi;
  const f16x2 bias = {(f16)1152.0f, (f16)1152.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = w[i] ^ 0x80808080u;
    const uint32_t x = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
    const uint32_t y = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
    if (i < 2) lo[2 * i] = x, lo[2 * i + 1] = y;
    else hi[2 * i - 4] = x, hi[2 * i - 3] = y;
  }
  a = __builtin_bit_cast(f16x8, lo);
  b = __builtin_bit_cast(f16x8, hi);
}

__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + kUnit - 1) / kUnit : 1; }

__device__ __forceinline__ int wave_sum_int(int v) {
  const int lane = lane_id();
#pragma unroll
  for (int x = 1; x < kWave; x *= 2) v += (int)from_lane((uint32_t)v, lane ^ x);
  return v;
}

template <int D, int NQ>
struct Shared {
  static constexpr int kCols = 16 * NQ;
  float o[kWaves][kCols][D + 4];
  float m[kWaves][kCols], l[kWaves][kCols];
  int last;
};

// One (sequence, key/value head, column block) over units [u0, u1) of its nu.
struct Segment {
  int b, head, cb, u0, u1, nu, len;
  int first_unit;  // of the whole pair, in the launch's numbering
  int pair;
};

template <int D, int NQ>
__device__ __forceinline__ void run_segment(const AttnArgs& a, const Segment& sg, int worker, int per_worker,
                                            Shared<D, NQ>& sh) {
  constexpr int KI = D / 64, VT = D / 16, COLS = 16 * NQ;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int len = sg.len, cols = a.new_tokens * a.group;
  const int t_begin = sg.u0 * kUnit, t_end = min(len, sg.u1 * kUnit);
  const int32_t* table = a.page_table + (int64_t)sg.b * a.table_stride;
  const int page_tokens = 1 << a.page_shift;

  // the query fragments, in the channel order of the key loads
  f16x8 qf[NQ][2 * KI];
  int limit[NQ];  // tokens the lane's column sees
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int col = sg.cb * COLS + 16 * n + r;
    const int i = col / a.group;
    limit[n] = col < cols ? len - a.new_tokens + i + 1 : 0;
    const uint16_t* row = a.q + ((int64_t)sg.b * a.new_tokens + i) * a.q_token +
                          (int64_t)(sg.head * a.group + (col - i * a.group)) * a.q_head;
#pragma unroll
    for (int k = 0; k < 2 * KI; ++k) {
      qf[n][k] = (f16x8)((f16)0.0f);
      if (col < cols) qf[n][k] = *reinterpret_cast<const f16x8*>(row + 64 * (k / 2) + 16 * g + 8 * (k & 1));
    }
  }

  // the largest value scale of the segment: the weights p * v_scale enter the
  // second product relative to it, as the sum of two fp16 numbers (one alone
  // would add as much error as the rounding of the output; the matrix cores are
  // idle most of the time here)
  float top = 0.0f;
  for (int p = (t_begin >> a.page_shift) + lane; p < (t_end + page_tokens - 1) >> a.page_shift; p += kWave) {
    const int id = table[p];
    if ((unsigned)id < (unsigned)a.num_pages) top = __builtin_fmaxf(top, a.v_scale[(int64_t)id * a.heads_kv + sg.head]);
  }
#pragma unroll
  for (int x = 1; x < kWave; x *= 2) top = __builtin_fmaxf(top, from_lane(top, lane ^ x));
  const int top_exp = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 0;

  f32x4 o[NQ][VT];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kNoMax, l[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < VT; ++d) o[n][d] = (f32x4)(0.0f);
  }

  for (int tb = t_begin + wave * kStep; tb < t_end; tb += kUnit) {
    // pages: the lane's own 16 tokens, and those of the key rows it loads
    const int tv = tb + 16 * g, tk = tb + 16 * (r >> 2);
    int pv = tv < len ? table[tv >> a.page_shift] : -1;
    int pk = tk < len ? table[tk >> a.page_shift] : -1;
    const bool held = (unsigned)pv < (unsigned)a.num_pages;
    if (!held) pv = 0;
    if ((unsigned)pk >= (unsigned)a.num_pages) pk = 0;
    const int64_t cv = (int64_t)pv * a.heads_kv + sg.head, ck = (int64_t)pk * a.heads_kv + sg.head;
    const float ks = held ? a.k_scale[cv] * a.scale : 0.0f;
    const float vs = held ? __builtin_amdgcn_ldexpf(a.v_scale[cv], kLift - top_exp) : 0.0f;
    const int8_t* kp = a.k_cache + ((ck << a.page_shift) + ((tk + (r & 3)) & (page_tokens - 1))) * D + 16 * g;
    const int8_t* vp = a.v_cache + ((cv * D + r) << a.page_shift) + (tv & (page_tokens - 1));
    u32x4 kw[4][KI], vw[VT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < KI; ++i) kw[t][i] = *reinterpret_cast<const u32x4*>(kp + t * 4 * D + i * 64);
#pragma unroll
    for (int d = 0; d < VT; ++d) vw[d] = *reinterpret_cast<const u32x4*>(vp + ((int64_t)(16 * d) << a.page_shift));

    f32x4 s[NQ][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][t] = (f32x4)(0.0f);
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        f16x8 x, y;
        codes_to_half(kw[t][i], x, y);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qf[n][2 * i], s[n][t], 0, 0, 0);
          s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, qf[n][2 * i + 1], s[n][t], 0, 0, 0);
        }
      }
    }
    f16x8 pf[NQ][2], pl[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float peak = kNoMax;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[n][t][i] * ks;
          if (!held || tv + 4 * t + i >= limit[n]) x = -__builtin_inff();
          s[n][t][i] = x;
          peak = __builtin_fmaxf(peak, x);
        }
      if (__any(peak > m[n] + kSlack)) {
        peak = __builtin_fmaxf(peak, from_lane(peak, lane ^ 16));
        peak = __builtin_fmaxf(peak, from_lane(peak, lane ^ 32));
        const float up = __builtin_fmaxf(peak, m[n]);
        const float f = __builtin_amdgcn_exp2f(m[n] - up);
        m[n] = up;
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < VT; ++d) o[n][d] *= f;
      }
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float p = __builtin_amdgcn_exp2f(s[n][2 * f + j / 4][j % 4] - m[n]);
          l[n] += p;
          const float w = p * vs;
          pf[n][f][j] = (f16)w;
          pl[n][f][j] = (f16)(w - (float)(f16)w);
        }
    }
#pragma unroll
    for (int d = 0; d < VT; ++d) {
      f16x8 x, y;
      codes_to_half(vw[d], x, y);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pf[n][0], o[n][d], 0, 0, 0);
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pf[n][1], o[n][d], 0, 0, 0);
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl[n][0], o[n][d], 0, 0, 0);
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pl[n][1], o[n][d], 0, 0, 0);
      }
    }
  }

  // the four waves' states -> one
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] += from_lane(l[n], lane ^ 16);
    l[n] += from_lane(l[n], lane ^ 32);
    if (g == 0) sh.m[wave][16 * n + r] = m[n], sh.l[wave][16 * n + r] = l[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int c = 16 * n + r;
    float up = kNoMax;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) up = __builtin_fmaxf(up, sh.m[w][c]);
    const float f = __builtin_amdgcn_exp2f(m[n] - up);
#pragma unroll
    for (int d = 0; d < VT; ++d) *reinterpret_cast<f32x4*>(&sh.o[wave][c][16 * d + 4 * g]) = o[n][d] * f;
  }
  __syncthreads();

  const bool whole = sg.u0 == 0 && sg.u1 == sg.nu;
  const int live = min(COLS, cols - sg.cb * COLS);  // columns of this block that exist
  // a worker's part of a pair that starts before its range, or of one that ends after it
  const int part_floats = COLS * (D + 2);
  float* part = a.parts + ((int64_t)worker * 2 + (sg.u0 > 0 ? 0 : 1)) * part_floats;
  for (int e = threadIdx.x; e < live * (D / 4); e += kWave * kWaves) {
    const int c = e / (D / 4), d = 4 * (e % (D / 4));
    float up = kNoMax, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) up = __builtin_fmaxf(up, sh.m[w][c]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += sh.l[w][c] * __builtin_amdgcn_exp2f(sh.m[w][c] - up);
    f32x4 x = (f32x4)(0.0f);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) x += *reinterpret_cast<const f32x4*>(&sh.o[w][c][d]);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_ldexpf(x[i], top_exp - kLift);
    if (whole) {
      const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
      const int col = sg.cb * COLS + c, i = col / a.group;
      uint16_t* row = a.out + ((int64_t)sg.b * a.new_tokens + i) * a.o_token +
                      (int64_t)(sg.head * a.group + (col - i * a.group)) * a.o_head + d;
      u32x2 w;
      w[0] = as_u32((f16x2){(f16)(x[0] * inv), (f16)(x[1] * inv)});
      w[1] = as_u32((f16x2){(f16)(x[2] * inv), (f16)(x[3] * inv)});
      *reinterpret_cast<u32x2*>(row) = w;
    } else {
      if (d == 0) publish(part + c, up), publish(part + COLS + c, sum);
#pragma unroll
      for (int i = 0; i < 4; ++i) publish(part + 2 * COLS + c * D + d + i, x[i]);
    }
  }
  if (whole) {
    __syncthreads();  // the next segment writes the shared states again
    return;
  }
  // the last of the pair's workers to arrive joins the parts, in worker order
  const int w_first = sg.first_unit / per_worker, w_last = (sg.first_unit + sg.nu - 1) / per_worker;
  wait_published();
  __syncthreads();
  if (threadIdx.x == 0) sh.last = arrive(a.counters + sg.pair) == w_last - w_first;
  __syncthreads();
  if (sh.last) {
    after_last_arrival();
    for (int e = threadIdx.x; e < live * (D / 4); e += kWave * kWaves) {
      const int c = e / (D / 4), d = 4 * (e % (D / 4));
      float up = kNoMax, sum = 0.0f;
      f32x4 x = (f32x4)(0.0f);
      for (int w = w_first; w <= w_last; ++w) {
        const bool starts_before = w * per_worker > sg.first_unit;
        const float* src = a.parts + ((int64_t)w * 2 + (starts_before ? 0 : 1)) * part_floats;
        const float pm = collect(src + c), pl = collect(src + COLS + c);
        f32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = collect(src + 2 * COLS + c * D + d + i);
        const float to = __builtin_fmaxf(up, pm);
        const float fx = __builtin_amdgcn_exp2f(up - to), fy = __builtin_amdgcn_exp2f(pm - to);
        up = to;
        sum = sum * fx + pl * fy;
        x = x * fx + y * fy;
      }
      const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
      const int col = sg.cb * COLS + c, i = col / a.group;
      uint16_t* row = a.out + ((int64_t)sg.b * a.new_tokens + i) * a.o_token +
                      (int64_t)(sg.head * a.group + (col - i * a.group)) * a.o_head + d;
      u32x2 wd;
      wd[0] = as_u32((f16x2){(f16)(x[0] * inv), (f16)(x[1] * inv)});
      wd[1] = as_u32((f16x2){(f16)(x[2] * inv), (f16)(x[3] * inv)});
      *reinterpret_cast<u32x2*>(row) = wd;
    }
    if (threadIdx.x == 0) reset_counter(a.counters + sg.pair);
  }
  __syncthreads();
}

// The launch's units, 256 tokens each, are numbered sequence by sequence, head
// by head, column block by column block; each workgroup takes an equal
// contiguous range of them, so ragged batches and single long sequences fill
// the chip alike.
template <int D, int NQ>
__global__ __launch_bounds__(kWave * kWaves) void kv8_attention_kernel(AttnArgs a) {
  __shared__ Shared<D, NQ> sh;
  const int lane = lane_id();
  const int pairs = a.heads_kv * a.col_blocks;
  int total = 0;
  for (int c = 0; c < a.batch; c += kWave)
    if (c + lane < a.batch) total += units_of(min(a.seq_lens[c + lane], a.max_tokens));
  total = __builtin_amdgcn_readfirstlane(wave_sum_int(total));
  const int units = total * pairs;
  const int per_worker = (units + gridDim.x - 1) / gridDim.x;
  const int worker = blockIdx.x;
  int u = worker * per_worker;
  const int u_end = min(units, u + per_worker);
  if (u >= u_end) return;
  // the sequence that holds unit u
  int b = 0, base = 0;
  for (int c = 0; c < a.batch; c += kWave) {
    const int mine = c + lane < a.batch ? units_of(min(a.seq_lens[c + lane], a.max_tokens)) * pairs : 0;
    int upto = mine;  // inclusive prefix sum
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) {
      const int o = (int)from_lane((uint32_t)upto, lane - x);
      if (lane >= x) upto += o;
    }
    const uint64_t past = __ballot(base + upto > u);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      b = c + at;
      base += __builtin_amdgcn_readlane(upto - mine, at);
      break;
    }
    base += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  while (u < u_end) {
    const int len = __builtin_amdgcn_readfirstlane(min(a.seq_lens[b], a.max_tokens));
    const int nu = units_of(len);
    const int seq_end = base + nu * pairs;
    while (u < min(u_end, seq_end)) {
      const int x = (u - base) / nu;
      Segment sg;
      sg.b = b, sg.head = x / a.col_blocks, sg.cb = x % a.col_blocks;
      sg.nu = nu, sg.len = max(len, 0), sg.first_unit = base + x * nu;
      sg.u0 = u - sg.first_unit, sg.u1 = min(nu, u_end - sg.first_unit);
      sg.pair = b * pairs + x;
      run_segment<D, NQ>(a, sg, worker, per_worker, sh);
      u = sg.first_unit + sg.u1;
    }
    base = seq_end;
    ++b;
  }
}

struct Plan {
  int nq, col_blocks;
  int64_t workers, counters;
  size_t scratch;
};

// Two workgroups a compute unit; fewer where the longest possible sequences
// hold fewer units.
Plan plan_of(int64_t batch, int64_t new_tokens, int64_t heads_q, int64_t heads_kv, int64_t head_dim,
             int64_t max_tokens) {
  Plan p;
  const int64_t cols = new_tokens * (heads_q / heads_kv);
  p.nq = cols > 16 ? 2 : 1;
  p.col_blocks = (int)((cols + 16 * p.nq - 1) / (16 * p.nq));
  const int64_t units = max_tokens > 0 ? (max_tokens + kUnit - 1) / kUnit : 1;
  p.counters = batch * heads_kv * p.col_blocks;
  const int64_t most = 2 * (int64_t)lbh::device_cus();
  p.workers = p.counters * units < most ? p.counters * units : most;
  p.scratch = ((size_t)p.workers * 2 * 16 * p.nq * (head_dim + 2) * 4 + 255) & ~(size_t)255;
  return p;
}

int check_sizes(int64_t batch, int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t head_dim,
                int64_t page_size, int64_t max_pages) {
  if (batch < 0 || tokens < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0 || max_pages < 0)
    return LB_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LB_ERR_PROB_SHAPE;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return LB_ERR_PROB_SHAPE;
  if (heads_q > 4096 || batch > (1 << 20) || tokens > (1 << 24) || max_pages > (1 << 28) / page_size) return LB_ERR_ARG;
  if (batch > 0 && tokens % batch != 0) return LB_ERR_ARG;
  if (batch > 0) {  // units and counters are numbered in 32 bits
    const int64_t cols = tokens / batch * (heads_q / heads_kv);
    const int64_t units = max_pages * page_size / kUnit + 1;
    if (batch * heads_kv * ((cols + 15) / 16) > (1 << 30) / units) return LB_ERR_PROB_SHAPE;
  }
  return LB_OK;
}

template <int D>
void launch(const AttnArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.workers), block(kWave * kWaves);
  if (p.nq == 1) kv8_attention_kernel<D, 1><<<grid, block, 0, st>>>(a);
  else kv8_attention_kernel<D, 2><<<grid, block, 0, st>>>(a);
}

}  // namespace
}  // namespace lb

extern "C" size_t lb_kv8_attention_scratch_bytes(int64_t batch, int64_t tokens, int64_t heads_q, int64_t heads_kv,
                                                 int64_t head_dim, int64_t page_size, int64_t max_pages) {
  if (lb::check_sizes(batch, tokens, heads_q, heads_kv, head_dim, page_size, max_pages) != LB_OK || batch == 0 ||
      tokens == 0)
    return 0;
  return lb::plan_of(batch, tokens / batch, heads_q, heads_kv, head_dim, page_size * max_pages).scratch;
}

extern "C" int lb_kv8_attention(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride,
                                const int8_t* k_cache, const int8_t* v_cache, const float* k_scale,
                                const float* v_scale, int64_t num_pages, int64_t page_size, const int32_t* page_table,
                                int64_t max_pages, int64_t table_stride, const int32_t* seq_lens, int64_t batch,
                                int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t head_dim, uint16_t* out,
                                int64_t o_token_stride, int64_t o_head_stride, float softmax_scale, int32_t* workspace,
                                int64_t workspace_len, void* scratch, size_t scratch_bytes, lb_stream_t stream) {
  using namespace lb;
  const int err = check_sizes(batch, tokens, heads_q, heads_kv, head_dim, page_size, max_pages);
  if (err != LB_OK) return err;
  if (num_pages < 0 || num_pages > 0x7fffffff || table_stride < max_pages) return LB_ERR_ARG;
  if (!(softmax_scale > 0.0f) || softmax_scale > 3e38f) return LB_ERR_ARG;
  if (batch == 0 || tokens == 0) return LB_OK;
  if (!q || !out || !seq_lens || !workspace) return LB_ERR_ARG;
  if (num_pages > 0 && max_pages > 0 && (!k_cache || !v_cache || !k_scale || !v_scale || !page_table)) return LB_ERR_ARG;
  const void* ptrs[] = {q, out, k_cache, v_cache, scratch};
  for (const void* p : ptrs)
    if (!lbh::aligned(p, 16)) return LB_ERR_ALIGN;
  if ((q_token_stride | q_head_stride | o_token_stride | o_head_stride) % 8 != 0) return LB_ERR_ALIGN;
  const Plan p = plan_of(batch, tokens / batch, heads_q, heads_kv, head_dim, page_size * max_pages);
  if (workspace_len < p.counters) return LB_ERR_WORKSPACE;
  if (scratch_bytes < p.scratch || !scratch) return LB_ERR_SCRATCH;

  AttnArgs a;
  a.q = q, a.q_token = q_token_stride, a.q_head = q_head_stride;
  a.k_cache = k_cache, a.v_cache = v_cache, a.k_scale = k_scale, a.v_scale = v_scale;
  a.page_table = page_table, a.seq_lens = seq_lens;
  a.out = out, a.o_token = o_token_stride, a.o_head = o_head_stride;
  a.counters = workspace, a.parts = static_cast<float*>(scratch);
  a.table_stride = table_stride, a.num_pages = (int)num_pages;
  a.page_shift = __builtin_ctzll((unsigned long long)page_size);
  // without pages no sequence holds a token
  a.max_tokens = num_pages > 0 ? (int)(max_pages * page_size) : 0;
  a.batch = (int)batch, a.new_tokens = (int)(tokens / batch), a.heads_kv = (int)heads_kv;
  a.group = (int)(heads_q / heads_kv), a.col_blocks = p.col_blocks;
  a.scale = softmax_scale * kLog2e;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (head_dim == 64) launch<64>(a, p, st);
  else if (head_dim == 128) launch<128>(a, p, st);
  else launch<256>(a, p, st);
  return lbh::launch_status();
}
