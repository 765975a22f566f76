// Causal attention inside each of the packed sequences of a batch of prompts.
//
//   o[i] = sum_{j <= i} softmax_j(scale q[i] . k[j]) v[j]      per sequence and query head
//
//   S^T = K Q^T    32x32x16: a lane holds 16 keys of one row, so a row's maximum
//                  and sum stay in the lane but for one exchange with lane ^ 32
//   O^T = V^T P^T  the weights of a lane are already the second product's operand
//
// The 128 rows of a workgroup are (token, query head of the group) pairs of one
// key/value head: a tile of 64 keys serves the whole group, the rows span few
// tokens, and little work falls past the diagonal.  Four waves of 32 rows go
// through the keys together, with the next tile on its way into LDS.
//
// Bound by the matrix cores at the clock that their load leaves (1.6 GHz of 2.4 at
// 128 channels), with LDS close behind: a product of 32 cycles reads 1 KB of keys or
// values, so four waves ask for all of the 128 bytes a cycle of a compute unit.  64
// rows a wave would halve that, but at 256 channels their accumulators, queries and
// scores do not fit the registers, and at 128 they leave one wave a SIMD, with
// nothing to run beside its softmax (8192 tokens: 920 us where 32 rows took 742).
//   8192 tokens, 40 / 8 heads of 128: 652 to 665 us, 1034 to 1054 TFLOP/s of the 1154
//   that a large library product reaches; 16384 tokens, 24 / 4 heads of 256: 3220 to
//   3310 us, 1000 to 1025 TFLOP/s; 8192 tokens, 32 / 8 heads of 64: 311 us, 884; 7
//   packed prompts of 100 to 1500 tokens, 24 / 4 heads of 256: 95 us, of which each
//   workgroup spends 7 on its first loads and its output.
#include "attn_common.hpp"

namespace lb {
namespace {

struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  const int32_t* starts;
  int batch, tokens, group, heads_kv, tiles;
  float scale;  // softmax scale * log2(e)
};

constexpr float kNoMax = -1e30f;
// The running maximum moves only when a score exceeds it by 2^kSlack, and the
// weights (and their sum) carry 2^kLift more: at most 2^15, inside fp16, and 2^7
// farther from its subnormals.
constexpr float kSlack = 8.0f, kLift = 7.0f;

typedef __attribute__((address_space(3))) void lds_void;
typedef __fp16 fp16x4 __attribute__((__vector_size__(8)));

// A weight is rounded to fp16 for the second product, its sum taken before that in
// fp32: an error of at most 2^-11 sum p |v|, as large as the output's own rounding
// where the values have one sign, and 2^-32 of the largest weight for one below
// fp16's normal numbers.  With normally distributed values the outputs are 2.7e-4
// (97 tokens: 2.2e-4) from exact, root mean square, where rounding them alone leaves
// 2.1e-4.  A second fp16 number for the rest, as over the cache, doubles that
// product: 8192 tokens, 128 channels, 664 -> 911 us, and no size has it for nothing
// (97 tokens 7.15 -> 7.75, 16 tokens 5.60 -> 5.87; 7 packed prompts of 256 channels
// 95 -> 115).

// Sixteen-byte chunks of a key (value) row change places so that the 16-byte
// reads of 16 rows at one column, and the transposing reads of 8 rows at one
// 64-byte column, use every bank.
template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  return D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
}

// A tile of keys (values) on its way into LDS, 16 bytes a lane and load, N loads
// a wave; rows past `rows` come out as zeros (the descriptor ends there).
template <int D, int KT, int W, bool KEYS>
struct Stage {
  static constexpr int N = KT * D / (W * kWave * 8);
  __amdgpu_buffer_rsrc_t from;
  __device__ __forceinline__ Stage(const uint16_t* base, int64_t token_stride, int rows)
      : from(buffer_of(base, rows > 0 ? (uint32_t)(((int64_t)(min(rows, KT) - 1) * token_stride + D) * 2) : 0u)) {}
  __device__ __forceinline__ void load(int j, int token_stride, uint16_t* lds, int wave, int lane) const {
    constexpr int C = D / 8;
    const int c = (j * W + wave) * kWave + lane;
    const int row = c / C, col = (c % C) ^ (KEYS ? k_swizzle<D>(row) : v_swizzle<D>(row));
    const uint32_t off = (uint32_t)(row * token_stride * 2 + col * 16);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)(lds + (j * W + wave) * kWave * 8), 16, off, 0, 0, 0);
  }
};

// The tiles with the most keys come first, whichever sequence they are of: a
// workgroup's time is its number of keys, and short ones last fill the ends (7
// packed prompts: 111 us, in the order of the sequences 133).
struct Place {
  int first, len, tile;  // of the sequence: its first token and length
};

struct Span {
  int first, len;
};
__device__ __forceinline__ Span span_of(const PromptArgs& a, int b) {
  if (b >= a.batch) return {0, 0};
  const int first = max(a.starts[b], 0);
  return {first, min(a.starts[b + 1], a.tokens) - first};
}
template <int ROWS>
__device__ __forceinline__ int tiles_of(const PromptArgs& a, int len) {
  return len > 0 ? (len * a.group + ROWS - 1) / ROWS : 0;
}

// Item i of all sequences' tiles in falling order of their place in the
// sequence; an empty place past the last.  64 sequences stay in registers.
template <int ROWS>
__device__ __forceinline__ Place place_of(const PromptArgs& a, int i) {
  const int lane = lane_id();
  const Span own = span_of(a, lane);
  const int own_tiles = tiles_of<ROWS>(a, own.len);
  auto from = [&](int t) {  // tiles at place t or later
    int n = __builtin_amdgcn_readlane(wave_scan(max(own_tiles - t, 0)), kWave - 1);
    for (int c = kWave; c < a.batch; c += kWave)
      n += __builtin_amdgcn_readlane(wave_scan(max(tiles_of<ROWS>(a, span_of(a, c + lane).len) - t, 0)), kWave - 1);
    return n;
  };
  int rank = from(0);
  if (rank <= i) return {0, 0, 0};
  int lo = rank - 1 - i;  // where one sequence has all the tiles
  if (a.batch > 1) {
    lo = 0;
    int hi = a.tiles;  // from(lo) > i >= from(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (from(mid) > i) lo = mid; else hi = mid;
    }
  }
  rank = i - from(lo + 1);  // among the sequences that have a tile lo
  for (int c = 0; c < a.batch; c += kWave) {
    const Span s = c ? span_of(a, c + lane) : own;
    const bool has = (c ? tiles_of<ROWS>(a, s.len) : own_tiles) > lo;
    const uint64_t m = __ballot(has);
    const int n = __popcll(m);
    if (rank < n) {
      const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
      const int at = __builtin_ctzll(__ballot(has && before == rank));
      return {__builtin_amdgcn_readlane(s.first, at), __builtin_amdgcn_readlane(s.len, at), lo};
    }
    rank -= n;
  }
  return {0, 0, 0};
}

// At 256 channels the output fills half of a wave's accumulation registers, which
// only the matrix products reach.  Without these marks (around the scaling, and at
// the end of the loop) the compiler copies all of it into vector registers in every
// tile, for the rare tile that scales it: 16384 tokens 3275 us, without 3470.
template <int D, int N>
__device__ __forceinline__ void stay_in_accumulators(f32x16 (&o)[N]) {
  if constexpr (D == 256)
#pragma unroll
    for (int d = 0; d < N; ++d) asm volatile("" : "+a"(o[d]));
}

template <int D, int KT, int W, int PER_SIMD>
__global__ __launch_bounds__(kWave * W, PER_SIMD) void prompt_attention_kernel(PromptArgs a) {
  constexpr int ROWS = W * 32, DT = D / 32, KK = D / 16, ST = KT / 32;
  // four arrays and not one: the compiler would make every read of a tile wait
  // for the loads of the next into the same array (16384 tokens: 3570 us, 4046)
  __shared__ __align__(16) uint16_t k0[KT * D], k1[KT * D], v0[KT * D], v1[KT * D];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.x % a.heads_kv, item = blockIdx.x / a.heads_kv;
  int first = 0, len = a.tokens, tile = a.tiles - 1 - item;
  if (a.starts != nullptr) {
    const Place at = place_of<ROWS>(a, item);
    first = at.first, len = at.len, tile = at.tile;
  }
  first = __builtin_amdgcn_readfirstlane(first), len = __builtin_amdgcn_readfirstlane(len);
  const int rows = len * a.group, row0 = tile * ROWS;
  if (row0 >= rows) return;
  const int last_token = (min(rows, row0 + ROWS) - 1) / a.group;
  const int tiles = last_token / KT + 1;
  const int wave_row = row0 + wave * 32;
  const int wave_first = wave_row / a.group;  // token of the wave's first row

  const int row = wave_row + r, token = row / a.group, head = kvh * a.group + row - token * a.group;
  const int seen = row < rows ? token : -1;  // the last key of the lane's row
  f16x8 qf[KK];
  {
    const uint16_t* p = a.q + (int64_t)(first + token) * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      qf[k] = (f16x8)((f16)0.0f);
      if (row < rows) qf[k] = *reinterpret_cast<const f16x8*>(p + 16 * k + 8 * h);
    }
  }
  const uint16_t* kbase = a.k + (int64_t)first * a.k_token + (int64_t)kvh * a.k_head;
  const uint16_t* vbase = a.v + (int64_t)first * a.v_token + (int64_t)kvh * a.v_head;

  f32x16 o[DT];
  float m = kNoMax, l = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = (f32x16)(0.0f);

  typedef Stage<D, KT, W, true> Keys;
  typedef Stage<D, KT, W, false> Values;
  static_assert(Keys::N + Values::N == KK, "one load of the next tile for each channel step of the scores");
  const int k_token = (int)a.k_token, v_token = (int)a.v_token;
  {
    const Keys keys(kbase, k_token, len);
    const Values values(vbase, v_token, len);
#pragma unroll
    for (int j = 0; j < Keys::N; ++j) keys.load(j, k_token, k0, wave, lane), values.load(j, v_token, v0, wave, lane);
  }
  // Tile kt from (kl, vl).  The next tile's loads into (kn, vn) go out between
  // the products of the scores: all at once they would hold up the wave (16
  // loads of 1 KB from four waves take 1000 cycles and more to be accepted).
  // After the last tile they have no rows: zeros, from nowhere.
  auto take = [&](int kt, const uint16_t* kl, const uint16_t* vl, uint16_t* kn, uint16_t* vn) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), as a builtin: the compiler then knows that the tile is there
    lds_barrier();
    const int64_t at = (int64_t)(kt + 1) * KT;
    const int left = kt + 1 < tiles ? len - (kt + 1) * KT : 0;
    const Keys keys(kbase + at * k_token, k_token, left);
    const Values values(vbase + at * v_token, v_token, left);
    auto load_next = [&](int j) {
      if (j < Keys::N) keys.load(j, k_token, kn, wave, lane);
      else values.load(j - Keys::N, v_token, vn, wave, lane);
    };
    f32x16 s[ST];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < ST; ++t) s[t] = (f32x16)(0.0f);
    constexpr int CH = KK / 4;  // channel steps of a quarter
    f16x8 kf[2][CH][ST];
    auto read_k = [&](int q) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int t = 0; t < ST; ++t) {
          const int row = 32 * t + r;
          kf[q & 1][k][t] = *reinterpret_cast<const f16x8*>(
              kl + row * D + 8 * ((2 * (q * CH + k) + h) ^ k_swizzle<D>(row)));
        }
    };
    read_k(0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q < 3) read_k(q + 1);
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int t = 0; t < ST; ++t)
          s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[q & 1][k][t], qf[q * CH + k], s[t], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < CH; ++k) load_next(q * CH + k);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (kt * KT + KT - 1 > wave_first) {
      const int past = seen - kt * KT - 4 * h;  // keys of the lane up to here are seen
#pragma unroll
      for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * t + 8 * (i >> 2) + (i & 3) > past) s[t][i] = -__builtin_inff();
    }
    float peak = kNoMax;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) peak = __builtin_fmaxf(peak, s[t][i]);
    peak *= a.scale;
    stay_in_accumulators<D>(o);
    if (__any(peak > m + kSlack)) {
      const float up = __builtin_fmaxf(__builtin_fmaxf(peak, from_lane(peak, lane ^ 32)), m);
      const float f = __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
      stay_in_accumulators<D>(o);
    }
    f16x8 pf[2 * ST];
    const float lift = kLift - m;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(s[t][i] * a.scale + lift);
        l += p;
        pf[2 * t + i / 8][i % 8] = (f16)p;
      }
#pragma unroll
    for (int c = 0; c < 2 * ST; ++c) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f16x8 vf;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int token = 16 * c + 8 * u + 4 * h + ((lane & 15) >> 2);
          const int chunk = (4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_swizzle<D>(token);
          const f16x4 x = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
              (__attribute__((address_space(3))) fp16x4*)(vl + token * D + 8 * chunk + 4 * (lane & 1))));
#pragma unroll
          for (int i = 0; i < 4; ++i) vf[4 * u + i] = x[i];
        }
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[c], o[d], 0, 0, 0);
      }
    }
  };
  for (int kt = 0; kt < tiles; kt += 2) {
    take(kt, k0, v0, k1, v1);
    if (kt + 1 < tiles) take(kt + 1, k1, v1, k0, v0);
    stay_in_accumulators<D>(o);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // no load may arrive in LDS after the workgroup

  // The rows leave through LDS (a wave's 32 x D in an array that no wave reads
  // any more): a store then takes whole rows, where a lane's accumulators are
  // four channels of a row each (97 tokens: 7.1 us, 7.9 without).  Chunks change
  // places as in the tiles.
  lds_barrier();
  uint16_t* mine = wave < 2 ? (wave == 0 ? k0 : k1) : (wave == 2 ? v0 : v1);
  static_assert(W == 4 && KT >= 32, "one array a wave");
  l += from_lane(l, lane ^ 32);
  const float inv = 1.0f / l;
  const int64_t place = (int64_t)(first + token) * a.o_token + (int64_t)head * a.o_head;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      u32x2 w;
      w[0] = as_u32((f16x2){(f16)(o[d][i] * inv), (f16)(o[d][i + 1] * inv)});
      w[1] = as_u32((f16x2){(f16)(o[d][i + 2] * inv), (f16)(o[d][i + 3] * inv)});
      const int chunk = (4 * d + i / 4) ^ k_swizzle<D>(r);
      *reinterpret_cast<u32x2*>(mine + r * D + 8 * chunk + 4 * h) = w;
    }
#pragma unroll
  for (int j = 0; j < 32 * D / 8 / kWave; ++j) {
    const int x = j * kWave + lane, rr = x / (D / 8), chunk = x % (D / 8);
    const uint32_t lo = from_lane((uint32_t)place, rr), hi = from_lane((uint32_t)(place >> 32), rr);
    const u32x4 w = *reinterpret_cast<const u32x4*>(mine + rr * D + 8 * (chunk ^ k_swizzle<D>(rr)));
    if (wave_row + rr < rows)
      *reinterpret_cast<u32x4*>(a.out + (int64_t)(((uint64_t)hi << 32) | lo) + 8 * chunk) = w;
  }
}

template <int D, int KT, int W, int PER_SIMD>
int launch(PromptArgs a, hipStream_t st) {
  constexpr int ROWS = W * 32;
  const int64_t rows = (int64_t)a.tokens * a.group;
  // every sequence may end inside a tile
  const int64_t tiles = a.starts ? rows / ROWS + a.batch : (rows + ROWS - 1) / ROWS;
  if (tiles * a.heads_kv > 0x7fffffff) return LB_ERR_PROB_SHAPE;
  a.tiles = (int)tiles;
  prompt_attention_kernel<D, KT, W, PER_SIMD><<<dim3((unsigned)(tiles * a.heads_kv)), dim3(kWave * W), 0, st>>>(a);
  return lbh::launch_status();
}

}  // namespace
}  // namespace lb

extern "C" int lb_prompt_attention(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, const uint16_t* k,
                                   int64_t k_token_stride, int64_t k_head_stride, const uint16_t* v,
                                   int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_seqlens,
                                   int64_t batch, int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t head_dim,
                                   uint16_t* out, int64_t o_token_stride, int64_t o_head_stride, float softmax_scale,
                                   lb_stream_t stream) {
  using namespace lb;
  if (batch < 0 || tokens < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0) return LB_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LB_ERR_PROB_SHAPE;
  if (heads_q > 4096 || batch > (1 << 20) || tokens > (1 << 26) || tokens * (heads_q / heads_kv) >= (1ll << 31) - 4096)
    return LB_ERR_ARG;
  if (!(softmax_scale > 0.0f) || softmax_scale > 3e38f) return LB_ERR_ARG;
  if (tokens == 0 || batch == 0) return LB_OK;
  if (cu_seqlens == nullptr && batch != 1) return LB_ERR_ARG;
  if (!q || !k || !v || !out) return LB_ERR_ARG;
  const void* ptrs[] = {q, k, v, out};
  for (const void* p : ptrs)
    if (!lbh::aligned(p, 16)) return LB_ERR_ALIGN;
  if ((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride |
       o_token_stride | o_head_stride) % 8 != 0)
    return LB_ERR_ALIGN;
  // a tile's offsets from its first key are 32-bit
  if (k_token_stride < 0 || v_token_stride < 0 || k_token_stride > (1 << 23) || v_token_stride > (1 << 23))
    return LB_ERR_ARG;
  PromptArgs a;
  a.q = q, a.k = k, a.v = v, a.out = out;
  a.q_token = q_token_stride, a.q_head = q_head_stride, a.k_token = k_token_stride, a.k_head = k_head_stride;
  a.v_token = v_token_stride, a.v_head = v_head_stride, a.o_token = o_token_stride, a.o_head = o_head_stride;
  a.starts = cu_seqlens, a.batch = (int)batch, a.tokens = (int)tokens, a.group = (int)(heads_q / heads_kv);
  a.heads_kv = (int)heads_kv, a.scale = softmax_scale * kLog2e;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // Waves a SIMD as the registers allow (142 of them, 220, 512): two workgroups a
  // compute unit, out of step by themselves, against one of eight waves at 128
  // channels: 691 us, 742.  Tiles of 32 keys at 256 channels: 4043 us, of 64: 3570.
  if (head_dim == 64) return launch<64, 64, 4, 3>(a, st);
  if (head_dim == 128) return launch<128, 64, 4, 2>(a, st);
  return launch<256, 64, 4, 1>(a, st);
}
