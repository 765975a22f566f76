// Attention of chunks of new tokens over the pages of the 8-bit cache: any number of
// new tokens a sequence, packed one after the other.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= len - n + i
//   k[j] = k_scale[page] ck[j],  v[j] = v_scale[page] cv[j]
//
//   S^T = K Q^T    32x32x16: a lane holds 32 keys of one row, so a row's maximum and
//                  sum stay in the lane but for one exchange with lane ^ 32
//   O^T = V^T P^T  the weights of a lane are already the second product's operand, and
//                  the value layout [channel][token] is its other one
//
// The 128 rows of a workgroup are (token, query head of the group) pairs of one
// key/value head.  Four waves of 32 rows go through tiles of 64 keys together: the
// codes of a tile come into registers while the tile before is computed, become fp16
// (exactly) and lie in LDS for all four.
//
// Bound by what a SIMD issues: of its cycles the products take half and vector instructions
// somewhat more (the codes to fp16 and the softmax in like shares), at the clock that the
// load leaves; LDS is busy half of them.  (4096 new tokens on 12288, 40 on 8 heads of 128:
// 1.22 ms, 986 TFLOP/s at 1.7 GHz.)  At 256 channels a SIMD has one wave, and 476 vector
// instructions of a tile stand beside 64 products: a third of the cycles each (2048 on 6144:
// 407 us, 887 TFLOP/s).  128 sequences of one new token: 161 us, 4.5 TB/s, where the operator
// for single tokens takes 122.  The smallest calls run instructions for the first time (24 on
// 301: 20 us, about 8 of them before the second tile and 4 for the second launch).
#include <algorithm>
#include <type_traits>

#include "attn_common.hpp"
#include "chunk_pieces.hpp"

namespace lb {
namespace {

// x / d for 0 <= x < 2^31 by a product: with 2^(s - 1) < d <= 2^s and m = ceil(2^(31 + s) / d)
// the product is off by less than x 2^s / 2^(31 + s) < 1 / d of a quotient.
struct Divisor {
  uint32_t m;
  int shift, d;
  explicit Divisor(int by = 1) : m(0), shift(0), d(by) {
    if (by <= 1) return;
    while ((1ll << (shift + 1)) < by) ++shift;
    m = (uint32_t)(((1ll << (32 + shift)) + by - 1) / by);
  }
  __device__ __forceinline__ int of(int x) const { return m ? (int)(__umulhi((uint32_t)x, m) >> shift) : x; }
};

struct ChunkArgs {
  const uint16_t* q;
  int64_t q_token, q_head;
  const int8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int32_t *page_table, *seq_lens, *starts;
  uint16_t* out;
  int64_t o_token, o_head;
  float* parts;
  struct Work* plan;  // behind the parts: how the keys were cut
  int64_t table_stride;
  int num_pages, page_shift, max_tokens, unit_shift;
  int batch, tokens;
  Divisor heads_kv, group;
  int workers, slots;  // workgroups that run at once; parts that the scratch holds
  float scale;         // softmax scale * log2(e)
};

constexpr int kRows = 128, kKeys = 1 << kTileShift, kWaves = 4;
constexpr float kNoMax = -1e30f;
// The running maximum is that of weight times value scale.  It moves only when
// exceeded by 2^kSlack, and the weights carry 2^kLift more: at most 2^15, inside
// fp16, and 2^7 farther from its subnormals.  A value scale is part of its weights'
// exponent, between 2^-kScales and 2^kScales (fp16 values give 2^-31 to 2^9), so that
// no weight that counts in the sum falls below fp32's normal numbers.
constexpr float kSlack = 8.0f, kLift = 7.0f, kScales = 32.0f, kMost = 32768.0f;  // 2^(kSlack + kLift)
// A piece of a row block's keys is this many tiles at least (with 8 or 16: 24 tokens on 301
// 25 and 32 us and not 20).
constexpr int kMinTiles = 2;
constexpr int kCuts = 24;
// In tiles: what a piece takes beside its own, the launch that joins cut ones, and for
// each round of these what their parts take to write and read.  (Pieces as long as the
// workers have on average: 7 of 17 to 900 tokens on up to 5000 311 us and not 243, two of up
// to 700 beside 40 single ones 234 and 191, 2048 on 6144 at 256 channels 535 and 461.)
constexpr float kPiece = 3.0f, kCut = 2.0f, kPart = 5.0f;
// Rounds of parts that the scratch holds (with six, and every row block cut: 4096 on 12288
// 1372 us and not 1348).
constexpr int kPartRounds = 4;

// Workgroups that run at once on a compute unit, a wave of each on a SIMD.  (256 channels
// fill the registers with one; 64 with three: 2048 on 2048 tokens 92.8 us and not 83.6.)
template <int D>
constexpr int kPerSimd = D == 256 ? 1 : 2;

// ------------------------------------------------------------- the work ---

// A sequence's new tokens begin at packed token `first`, position `at` (below 0 for
// padding); the table holds its first `len` tokens.
struct Seq {
  int first, n, len, at;
};
__device__ __forceinline__ Seq seq_of(const ChunkArgs& a, int b) {
  if (b >= a.batch) return {0, 0, 0, 0};
  Seq s;
  s.first = max(a.starts[b], 0);
  s.n = max(min(a.starts[b + 1], a.tokens) - s.first, 0);
  const int full = max(a.seq_lens[b], 0);
  s.len = min(full, a.max_tokens), s.at = full - s.n;
  return s;
}
__device__ __forceinline__ int blocks_of(const ChunkArgs& a, const Seq& s) { return (s.n * a.group.d + kRows - 1) / kRows; }
// What the keys of a sequence are cut by: tiles, or units of a few in the longest tables.
__device__ __forceinline__ int tiles_of(const ChunkArgs& a, const Seq& s) { return max(units_of(s.len, a.unit_shift), 1); }
// Up to kSorted sequences' row blocks and tiles stay in registers, lane l those of sequence
// 64 c + l.
constexpr int kChunks = 4, kSorted = kChunks * kWave;
struct Sizes {
  Seq own;  // of the first 64
  int blocks[kChunks], tiles[kChunks];
};
__device__ __forceinline__ Sizes sizes_of(const ChunkArgs& a) {
  Sizes z;
  z.own = seq_of(a, lane_id());
  z.blocks[0] = blocks_of(a, z.own), z.tiles[0] = tiles_of(a, z.own);
#pragma unroll
  for (int c = 1; c < kChunks; ++c) {
    z.blocks[c] = 0, z.tiles[c] = 1;
    if (c * kWave >= a.batch || a.batch > kSorted) continue;
    const Seq s = seq_of(a, c * kWave + lane_id());
    z.blocks[c] = blocks_of(a, s), z.tiles[c] = tiles_of(a, s);
  }
  return z;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), kWave - 1); }
// The lane with the smallest v (above zero), the lowest of several.
__device__ __forceinline__ int wave_least(float v) {
  uint32_t x = (__builtin_bit_cast(uint32_t, v) & ~63u) | lane_id();
  auto least = [&](uint32_t other) { x = min(x, other); };
  least(__builtin_amdgcn_update_dpp(~0, x, 0x111, 0xf, 0xf, false));  // as in wave_scan
  least(__builtin_amdgcn_update_dpp(~0, x, 0x112, 0xf, 0xf, false));
  least(__builtin_amdgcn_update_dpp(~0, x, 0x114, 0xf, 0xf, false));
  least(__builtin_amdgcn_update_dpp(~0, x, 0x118, 0xf, 0xf, false));
  least(__builtin_amdgcn_update_dpp(~0, x, 0x142, 0xa, 0xf, false));
  least(__builtin_amdgcn_update_dpp(~0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, kWave - 1) & 63;
}

// Every row block's keys are cut into pieces of at most `most` tiles, a workgroup each.
struct Work {
  int most, total;  // pieces of all sequences, of one head
  int tail, cuts;   // of a single sequence: so many first row blocks are cut into `cuts`, the others not at all (tail 0: all alike)
};
// A lane tries one length of the pieces: the longest row block's keys cut into one to
// kCuts, or what all workers have in all and somewhat more, so that all run at once.  What
// has the least rounds of pieces times their mean length, and the time that a piece takes
// besides, is taken.  (Above 64 sequences: what the workers have in all.)
__device__ __forceinline__ Work work_of(const ChunkArgs& a, const Sizes& z) {
  const int lane = lane_id(), blocks = z.blocks[0], tiles = z.tiles[0];
  const float heads = (float)a.heads_kv.d, slots = __builtin_amdgcn_rcpf((float)a.workers);
  if (a.batch > kWave && a.batch <= kSorted) {
    int all = 0, n = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) all += z.blocks[c] * z.tiles[c];
    const int most = max(min((int)((float)wave_total(all) * heads * slots) + 1, kMostUnits), kMinTiles);
    const float inverse = __builtin_amdgcn_rcpf((float)most);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) n += z.blocks[c] * pieces_in(z.tiles[c], most, inverse);
    return {most, wave_total(n), 0, 1};
  }
  if (a.batch > kWave) {
    int all = wave_total(blocks * tiles);
    for (int c = kWave; c < a.batch; c += kWave) {
      const Seq s = seq_of(a, c + lane);
      all += wave_total(blocks_of(a, s) * tiles_of(a, s));
    }
    const int most = max(min((int)((float)all * heads * slots) + 1, kMostUnits), kMinTiles);
    const float inverse = __builtin_amdgcn_rcpf((float)most);
    int n = wave_total(blocks * pieces_in(tiles, most, inverse));
    for (int c = kWave; c < a.batch; c += kWave) {
      const Seq s = seq_of(a, c + lane);
      n += wave_total(blocks_of(a, s) * pieces_in(tiles_of(a, s), most, inverse));
    }
    return {most, n, 0, 1};
  }
  int all = 0, longest = 1;
  for (int b = 0; b < a.batch; ++b) {
    const int n = __builtin_amdgcn_readlane(blocks, b), t = __builtin_amdgcn_readlane(tiles, b);
    all += n * t;
    if (n) longest = max(longest, t);
  }
  const float work = (float)all * heads, share = work * slots;
  const int cuts = lane + 1;
  int most = lane < kCuts ? (int)((float)(longest + lane) * __builtin_amdgcn_rcpf((float)cuts) + 0.5f) : (int)(share * (1.0f + (lane - kCuts) * 0.02f)) + 1;
  most = max(min(most, longest), kMinTiles);
  const float inverse = __builtin_amdgcn_rcpf((float)most);
  int n = 0, cut = 0;
  for (int b = 0; b < a.batch; ++b) {
    const int each = pieces_in(__builtin_amdgcn_readlane(tiles, b), most, inverse), x = __builtin_amdgcn_readlane(blocks, b) * each;
    n += x, cut += each > 1 ? x : 0;
  }
  const float count = (float)n * heads, rounds = __builtin_ceilf(count * slots);
  const float mean = __builtin_fmaxf(work * __builtin_amdgcn_rcpf(count), rounds <= 1.0f ? (float)min(most, longest) : 0.0f);
  float cost = rounds * (mean + kPiece);
  if (cut) cost += kCut + kPart * (float)cut * heads * slots;
  if (cut * a.heads_kv.d > a.slots) cost = 3e38f;
  const int best = wave_least(cost);
  Work w = {__builtin_amdgcn_readlane(most, best), __builtin_amdgcn_readlane(n, best), 0, 1};
  if (a.batch == 1) {
    // whole row blocks for some rounds, and what is left of them, the shortest, cut so that it
    // fills one more (2048 on 14336 711 us and not 742, 4096 on 12288 1296 and not 1398)
    const int count = __builtin_amdgcn_readlane(blocks, 0), full = (int)((float)(count * a.heads_kv.d) * slots + 0.001f);
    const int tail = count - (int)((float)(full * a.workers) * __builtin_amdgcn_rcpf(heads) + 0.001f);
    const int cuts = tail > 0 ? (int)((float)a.workers * __builtin_amdgcn_rcpf((float)tail * heads) + 0.001f) : 1;
    const float least = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, cost), best));
    const float one = (float)longest, tailed = (float)full * (one + kPiece) + one * __builtin_amdgcn_rcpf((float)cuts) + kPiece + kCut + kPart;
    if (full > 0 && cuts > 1 && longest >= cuts * kMinTiles && tail * cuts * a.heads_kv.d <= a.slots && tailed < least)
      w = {longest, count - tail + tail * cuts, tail, cuts};
  }
  return w;
}

// A row block's piece of keys, tiles [t0, t1).
struct Piece {
  int b, block, pieces, piece, t0, t1;
  int slot;  // among the pieces of all split row blocks of one head
  Seq s;
};
__device__ __forceinline__ int block_tiles(const ChunkArgs& a, const Seq& s, int block) {
  const int last = min(s.n - 1, a.group.of((block + 1) * kRows - 1));  // token of the last row
  return max((min(s.at + last + 1, s.len) + kKeys - 1) / kKeys, 0);
}
__device__ __forceinline__ Seq seq_from(const Seq& s, int lane) {
  return {__builtin_amdgcn_readlane(s.first, lane), __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.len, lane),
          __builtin_amdgcn_readlane(s.at, lane)};
}
// Piece i of all, the last row block of a sequence first.  With more pieces than run at
// once the sequences with the longest come first (of up to kSorted): short ones last fill
// the ends (128 decoding sequences of 500 to 8192 tokens, 8 heads of 128: 161 us, and 193 in
// the order of the sequences; three of up to 500 new tokens beside 200 single ones 222 and
// 248).
// JOIN: row block i of those that have several pieces, and its first.
template <bool JOIN>
__device__ __forceinline__ bool piece_of(const ChunkArgs& a, const Sizes& z, const Work& w, int i, Piece& p) {
  const int lane = lane_id();
  const Seq& own = z.own;
  const float inverse = __builtin_amdgcn_rcpf((float)w.most);
  // x-th piece (row block) of the sequence in lane `at`, which has `blocks` cut into `pieces`
  auto found = [&](const Seq& s, int b, int at, int x, int blocks, int pieces, int slots) {
    p.s = seq_from(s, at), p.b = b, p.pieces = pieces;
    int q = JOIN ? x : (int)(((float)x + 0.5f) * __builtin_amdgcn_rcpf((float)pieces));
    p.piece = JOIN ? 0 : x - q * pieces;
    if (!JOIN && p.piece < 0) --q, p.piece += pieces;
    if (!JOIN && p.piece >= pieces) ++q, p.piece -= pieces;
    p.block = blocks - 1 - q;
    p.slot = slots + q * pieces + p.piece;
    const int tiles = block_tiles(a, p.s, p.block);
    const float each = (float)tiles * __builtin_amdgcn_rcpf((float)pieces);
    p.t0 = min((int)(each * (float)p.piece), tiles);
    p.t1 = p.piece + 1 == pieces ? tiles : min((int)(each * (float)(p.piece + 1)), tiles);
  };
  if (a.batch == 1) {
    const int blocks = __builtin_amdgcn_readlane(z.blocks[0], 0);
    if (w.tail) {
      const int whole = blocks - w.tail;
      if (i >= (JOIN ? w.tail : w.total)) return false;
      if (JOIN) found(own, 0, 0, i, w.tail, w.cuts, 0);
      else if (i < whole) found(own, 0, 0, i, blocks, 1, 0);
      else found(own, 0, 0, i - whole, w.tail, w.cuts, 0);
      return true;
    }
    const int pieces = __builtin_amdgcn_readlane(pieces_in(z.tiles[0], w.most, inverse), 0);
    if (i >= (JOIN ? (pieces > 1 ? blocks : 0) : blocks * pieces)) return false;
    found(own, 0, 0, i, blocks, pieces, 0);
    return true;
  }
  int slots = 0;
  if (a.batch <= kSorted) {
    int pieces[kChunks], size[kChunks], length[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      pieces[c] = pieces_in(z.tiles[c], w.most, inverse);
      size[c] = JOIN ? (pieces[c] > 1 ? z.blocks[c] : 0) : z.blocks[c] * pieces[c];
      length[c] = pieces[c] > 1 ? w.most : z.tiles[c];  // at most w.most
    }
    auto from = [&](int t) {  // pieces of t tiles or more
      int n = 0;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) n += length[c] >= t ? size[c] : 0;
      return wave_total(n);
    };
    int lo = 0;
    if (!JOIN && w.total * a.heads_kv.d > a.workers) {
      if (i >= w.total) return false;
      lo = 1;
      int hi = w.most + 1;  // from(lo) > i >= from(hi)
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (from(mid) > i) lo = mid; else hi = mid;
      }
      i -= from(lo + 1);
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (c * kWave >= a.batch) break;
      const int mine = lo == 0 || length[c] == lo ? size[c] : 0;
      const int upto = wave_scan(mine), all = __builtin_amdgcn_readlane(upto, kWave - 1);
      const int split = pieces[c] > 1 ? z.blocks[c] * pieces[c] : 0, split_upto = wave_scan(split);
      if (i < all) {
        const int at = __builtin_ctzll(__ballot(upto > i));
        const Seq s = c ? seq_of(a, c * kWave + lane) : own;
        found(s, c * kWave + at, at, i - __builtin_amdgcn_readlane(upto - mine, at), __builtin_amdgcn_readlane(z.blocks[c], at),
              __builtin_amdgcn_readlane(pieces[c], at), slots + __builtin_amdgcn_readlane(split_upto - split, at));
        return true;
      }
      i -= all, slots += __builtin_amdgcn_readlane(split_upto, kWave - 1);
    }
    return false;
  }
  int base = 0;
  for (int c = 0; c < a.batch; c += kWave) {
    const Seq s = c ? seq_of(a, c + lane) : own;
    const int blocks = blocks_of(a, s), pieces = pieces_in(tiles_of(a, s), w.most, inverse);
    const int split = pieces > 1 ? blocks * pieces : 0;
    const int size = JOIN ? (pieces > 1 ? blocks : 0) : blocks * pieces;
    const int upto = wave_scan(size), all = __builtin_amdgcn_readlane(upto, kWave - 1);
    const int split_upto = wave_scan(split);
    if (base + all > i) {
      const int at = __builtin_ctzll(__ballot(base + upto > i));
      found(s, c + at, at, i - base - __builtin_amdgcn_readlane(upto - size, at), __builtin_amdgcn_readlane(blocks, at),
            __builtin_amdgcn_readlane(pieces, at), slots + __builtin_amdgcn_readlane(split_upto - split, at));
      return true;
    }
    base += all, slots += __builtin_amdgcn_readlane(split_upto, kWave - 1);
  }
  return false;
}

// A part: the rows' maxima and sums, then each wave's accumulators as its lanes hold
// them, sixteen bytes a lane side by side.
template <int D>
constexpr int kPartFloats = kRows * (D + 2);

// ------------------------------------------------------------- a tile ---

// The 16-byte chunks of a key's row change places so that reads use every bank: of the
// keys 0 to 3 and 16 to 19 and so on, which the lanes of a product's operand read.
template <int D>
__device__ __forceinline__ int k_swizzle(int key) {
  const int b2 = key >> 2 & 1, b4 = key >> 4 & 1;
  return D == 64 ? (key >> 1 & 1) | b4 << 1 | b2 << 2 : (key & 3) | b4 << 2 | b2 << 3;
}

// Sixteen tiles' pages and scales are looked up together (4096 on 12288 1267 us, and 1300 with
// a tile's at a time), lane l those of the 16 tokens l % 4 of tile l / 4, and what the products
// need of them lies in LDS for all waves: the factor of the scores, the value scale as an
// exponent, the inverse of that (2^-kLift times), and what is left of a value scale outside
// the exponent's range.
constexpr int kBatch = 16;
typedef f32x4 Info[2][kBatch * 4];

// The tiles of a piece on their way: pages and scales a batch ahead, codes DEPTH tiles.
template <int D, int DEPTH>
struct Tiles {
  static constexpr int N = D / 64;  // loads of keys (and of values) of a thread and tile
  const ChunkArgs& a;
  Info& info;
  const int32_t* table;
  int head, len, first, lane, wave;
  int groups;     // log2 of the groups of 16 tokens, of a tile's four, that lie side by side in a page
  int per, in;    // channels of a load of values, loads of all channels
  uint32_t k_off, v_off;  // the thread's place in a load
  int k_lds, v_lds[N];    // and in LDS
  uint32_t k_at[2], v_at[2];  // lane l: where the codes of its 16 tokens are, of the batch that is loaded
  int cell, page;             // page and head, of the next batch; page of the one after
  float ks, vs;               // scales of the next batch
  uint64_t held, odd, next_held, next_odd;  // bit l: page there; scales not finite, not above zero or outside the range
  uint64_t strange;                         // bit 4 i: tile i has a group without a page, or odd
  u32x4 codes[DEPTH][2 * N];

  __device__ __forceinline__ Tiles(const ChunkArgs& args, Info& shared, const Piece& p, int kv_head, int w)
      : a(args), info(shared), head(kv_head), len(p.s.len), first(p.t0), lane(lane_id()), wave(w) {
    table = a.page_table + (int64_t)p.b * a.table_stride;
    groups = min(a.page_shift - 4, 2), per = kWave >> groups, in = D / per;
    const int row = (wave * kWave + lane) / (D / 16), col = 2 * (lane % (D / 16));
    k_off = (row & 15) * D + col * 8;
    k_lds = row * D + 8 * (col ^ (col >> 4) ^ k_swizzle<D>(row));
    v_off = (((wave % in) * per + (lane >> groups)) << a.page_shift) + (lane & ((1 << groups) - 1)) * 16;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int y = i * kWaves + wave, g = (y / in << groups) + (lane & ((1 << groups) - 1));
      const int ch = (y % in) * per + (lane >> groups);
      v_lds[i] = ch * kKeys + 8 * ((2 * g) ^ (ch >> 1 & 7));
    }
  }
  __device__ __forceinline__ int token(int batch) const { return (first + batch * kBatch) * kKeys + 16 * lane; }
  __device__ __forceinline__ void load_pages(int batch) { page = table[min(token(batch), len - 1) >> a.page_shift]; }
  __device__ __forceinline__ void load_scales(int batch) {
    const bool real = token(batch) < len && (unsigned)page < (unsigned)a.num_pages;
    next_held = __ballot(real);
    cell = (real ? page : 0) * a.heads_kv.d + head;
    ks = a.k_scale[cell], vs = a.v_scale[cell];
  }
  __device__ __forceinline__ void tell(int batch) {
    const bool real = next_held >> lane & 1;
    const float v = real ? vs : 1.0f;
    // a scale of infinity has no scores: ks - ks makes it NaN and is zero otherwise
    const float k = real ? ks * a.scale + (ks - ks) : 1.0f;
    const float lg = __builtin_fmaxf(__builtin_fminf(__builtin_amdgcn_logf(__builtin_fabsf(v)), kScales), -kScales);
    next_odd = __ballot(!(k > 0.0f && k < __builtin_inff() && v > 0.0f && __builtin_fabsf(lg) < kScales));
    if (lane / kBatch == wave) info[batch & 1][lane] = (f32x4){k, lg, __builtin_amdgcn_exp2f(-lg - kLift), v * __builtin_amdgcn_exp2f(-lg)};
  }
  __device__ __forceinline__ void turn() {
    held = next_held, odd = next_odd;
    strange = ~held | odd;
    strange |= strange >> 1;
    strange |= strange >> 2;
  }
  __device__ __forceinline__ void locate(int batch) {
    const int in_page = token(batch) & ((1 << a.page_shift) - 1);
    const uint64_t k = (uint64_t)(uintptr_t)a.k_cache + (uint64_t)((((int64_t)cell << a.page_shift) + in_page) * D);
    const uint64_t v = (uint64_t)(uintptr_t)a.v_cache + (uint64_t)(((int64_t)cell * D << a.page_shift) + in_page);
    k_at[0] = (uint32_t)k, k_at[1] = (uint32_t)(k >> 32), v_at[0] = (uint32_t)v, v_at[1] = (uint32_t)(v >> 32);
  }
  // Tile i of the piece is about to be computed, the loads of tile i + 1 + DEPTH to be sent
  // off.  A batch's places in LDS are written at least a barrier after their last readers.
  __device__ __forceinline__ void step(int i) {
    const int c = i % kBatch, batch = i / kBatch;
    if (c == kBatch - 1 - DEPTH) locate(batch + 1);
    if (i % 2) return;
    if (c == 0 && i > 0) turn();
    else if (c == 2) load_scales(batch + 1);
    else if (c == 8) tell(batch + 1);
  }
  // After the last use of the pages' numbers: the batch after the next one's.
  __device__ __forceinline__ void step_after(int i) {
    if (i % kBatch == 4) load_pages(i / kBatch + 2);
  }
  // Load j of tile i: of its keys, then of its values; none of one that is not `real`.
  __device__ __forceinline__ void load(int set, int j, int i, bool real) {
    const int at_lane = i % kBatch * 4;
    const int y = (j - N) * kWaves + wave;
    const int l = at_lane + (j < N ? (j * kWaves + wave) * (kWave * 16 / D) / 16 : y / in << groups);  // the load's 16 tokens
    const uint32_t* at = j < N ? k_at : v_at;
    const uint64_t base = (uint32_t)__builtin_amdgcn_readlane(at[0], l) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at[1], l) << 32;
    const uint32_t bytes = real ? (uint32_t)D << a.page_shift : 0u;
    codes[set][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
        buffer_of(reinterpret_cast<const void*>(base), bytes), j < N ? k_off : v_off, j < N ? 0 : ((j - N) * kWaves % in * per) << a.page_shift, 0));
  }
  // As fp16 into LDS: keys [token][channel], values [channel][token].
  __device__ __forceinline__ void store(int set, int j, uint16_t* kl, uint16_t* vl) const {
    f16x8 x, y;
    codes_to_half(codes[set][j], x, y);
    if (j < N) {
      constexpr int kRowStep = kWaves * kWave / (D / 16);
      static_assert(N == 1 || kRowStep == 32 || kRowStep == 16, "the rows of a thread's loads change places alike, or as 16 says");
      const int at = k_lds ^ (kRowStep == 16 && (j & 1) ? 8 << 2 : 0);
      *reinterpret_cast<f16x8*>(kl + at + j * kRowStep * D) = x;
      *reinterpret_cast<f16x8*>(kl + (at ^ 8) + j * kRowStep * D) = y;
    } else {
      *reinterpret_cast<f16x8*>(vl + v_lds[j - N]) = x;
      *reinterpret_cast<f16x8*>(vl + (v_lds[j - N] ^ 8)) = y;
    }
  }
};

// At 256 channels the output fills half of a wave's accumulation registers, which only
// the matrix products reach; without these marks the compiler copies all of it into
// vector registers in every tile, for the rare tile that scales it.
template <int D, int N>
__device__ __forceinline__ void stay_in_accumulators(f32x16 (&o)[N]) {
  if constexpr (D == 256)
#pragma unroll
    for (int d = 0; d < N; ++d) asm volatile("" : "+a"(o[d]));
}

// The end of a piece of up to 32 rows: waves 0 and 1 hold the first half of the channels,
// of 32 keys of every tile each, 2 and 3 the second.  `sums` (fp16 of 32 rows and more),
// `states` and `lines` are places in LDS that no wave reads any more after a barrier.
template <int D, int N>
__device__ __forceinline__ void finish_thin(const ChunkArgs& a, const Piece& p, int kvh, int wave, int lane, f32x16 (&o)[N], float m, float l,
                                            uint16_t* sums, float* states, uint16_t* lines) {
  constexpr int DB = D / 64;
  const int r = lane & 31, h = lane >> 5, half = wave >> 1, rows = p.s.n * a.group.d, first = p.block * kRows;
  f32x4* to = reinterpret_cast<f32x4*>(sums) + lane;
  lds_barrier();
  if (wave & 1) {
    if (h == 0) states[half * 64 + r] = m, states[half * 64 + 32 + r] = l;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) to[(4 * d + i) * kWave] = (f32x4){o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
  }
  lds_barrier();
  if (!(wave & 1)) {
    const float m1 = states[half * 64 + r], l1 = states[half * 64 + 32 + r], up = __builtin_fmaxf(m, m1);
    const float f = __builtin_amdgcn_exp2f(m - up), f1 = __builtin_amdgcn_exp2f(m1 - up);
    m = up, l = l * f + l1 * f1;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 x = to[(4 * d + i) * kWave];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][4 * i + j] = o[d][4 * i + j] * f + x[j] * f1;
      }
  }
  if (p.pieces > 1) {
    const int slot = p.slot * a.heads_kv.d + kvh;
    if (slot >= a.slots || (wave & 1) || first + r >= rows) return;
    float* part = a.parts + (int64_t)slot * kPartFloats<D>;
    if (lane == r && half == 0) part[r] = m, part[kRows + r] = l;
    f32x4* out = reinterpret_cast<f32x4*>(part + 2 * kRows) + lane;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) out[(4 * (half * DB + d) + i) * kWave] = (f32x4){o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    return;
  }
  if (!(wave & 1)) {
    const float inv = l > 0.0f ? __builtin_exp2f(-kLift) / l : l == 0.0f ? 0.0f : l;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        u32x2 w;
        w[0] = as_u32((f16x2){(f16)(o[d][i] * inv), (f16)(o[d][i + 1] * inv)});
        w[1] = as_u32((f16x2){(f16)(o[d][i + 2] * inv), (f16)(o[d][i + 3] * inv)});
        *reinterpret_cast<u32x2*>(lines + r * D + 8 * ((4 * (half * DB + d) + i / 4) ^ k_swizzle<D>(r)) + 4 * h) = w;
      }
  }
  lds_barrier();
#pragma unroll
  for (int j = 0; j < 32 * D / 8 / (kWave * kWaves); ++j) {
    const int x = (j * kWaves + wave) * kWave + lane, rr = x / (D / 8), chunk = x % (D / 8);
    const int row = first + rr, token = a.group.of(row), head = kvh * a.group.d + row - token * a.group.d;
    const u32x4 w = *reinterpret_cast<const u32x4*>(lines + rr * D + 8 * (chunk ^ k_swizzle<D>(rr)));
    if (row < rows) *reinterpret_cast<u32x4*>(a.out + (int64_t)(p.s.first + token) * a.o_token + (int64_t)head * a.o_head + 8 * chunk) = w;
  }
}

// The end of a piece of more rows: each wave's 32, through `mine`, where no wave reads any
// more after a barrier.  (The row's place is found once more: kept over the loop it would
// take registers.)
template <int D, int N>
__device__ __forceinline__ void finish(const ChunkArgs& a, const Piece& p, int kvh, int wave, int lane, f32x16 (&o)[N], float m, float l, uint16_t* mine) {
  constexpr int DT = D / 32;
  const int r = lane & 31, h = lane >> 5, rows = p.s.n * a.group.d, wave_row = p.block * kRows + wave * 32;
  int row = wave_row + r;
  asm volatile("" : "+v"(row));
  if (p.pieces > 1) {
    const int slot = p.slot * a.heads_kv.d + kvh;
    if (slot >= a.slots) return;
    float* part = a.parts + (int64_t)slot * kPartFloats<D>;
    if (row < rows) {
      if (h == 0) part[wave * 32 + r] = m, part[kRows + wave * 32 + r] = l;
      f32x4* to = reinterpret_cast<f32x4*>(part + 2 * kRows + wave * 32 * D) + lane;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          to[(4 * d + i) * kWave] = (f32x4){o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    }
    return;
  }
  // the rows leave through LDS, a wave's 32 x D in an array that no wave reads any more
  lds_barrier();
  const float inv = l > 0.0f ? __builtin_exp2f(-kLift) / l : l == 0.0f ? 0.0f : l;
  const int to_token = a.group.of(row), to_head = kvh * a.group.d + row - to_token * a.group.d;
  const int64_t place = (int64_t)(p.s.first + to_token) * a.o_token + (int64_t)to_head * a.o_head;
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

// A piece, by the waves of a workgroup.  THIN: a row block of up to 32 rows, which the waves
// share: each takes half of the keys and half of the channels (two of up to 700 tokens beside
// 40 single ones 173 us, and 203 with the rows in one wave; 128 single ones 205 and 237).
template <int D, bool THIN>
__device__ __forceinline__ void run(const ChunkArgs& a, const Piece& p, int kvh, uint16_t* k0, uint16_t* k1, uint16_t* v0, uint16_t* v1, Info& info) {
  constexpr int DT = D / 32, KK = D / 16, ST = kKeys / 32, OB = THIN ? DT / 2 : DT;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 31, h = lane >> 5;
  const int rows = p.s.n * a.group.d;
  const int wave_row = p.block * kRows + (THIN ? 0 : wave * 32);
  const int row = wave_row + r, token = a.group.of(row), q_head = kvh * a.group.d + row - token * a.group.d;
  const bool real = row < rows;
  // the lane's row sees the keys up to `seen`, all of the wave's those up to `all_see`
  const int seen = real ? min(p.s.at + token, p.s.len - 1) : -1;
  const int all_see = min(p.s.at + a.group.of(wave_row), p.s.len - 1);

  f16x8 qf[KK];
  {
    const uint16_t* from = a.q + (int64_t)(p.s.first + token) * a.q_token + (int64_t)q_head * a.q_head;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      qf[k] = (f16x8)((f16)0.0f);
      if (real) qf[k] = *reinterpret_cast<const f16x8*>(from + 16 * k + 8 * h);
    }
  }
  f32x16 o[OB];
  float m = kNoMax, l = 0.0f;
#pragma unroll
  for (int d = 0; d < OB; ++d) o[d] = (f32x16)(0.0f);

  // a thin block's tile is done before the next one's codes can arrive; it has registers
  // to spare (7 of 17 to 900 tokens 224 us, and 247 a tile ahead)
  constexpr int DEPTH = THIN ? 2 : 1;
  typedef Tiles<D, DEPTH> T;
  T tiles(a, info, p, kvh, wave);
  const int count = p.t1 - p.t0;
  if (count > 0) {
    tiles.load_pages(0);
    tiles.load_scales(0);
    tiles.locate(0);
    tiles.load_pages(1);
#pragma unroll
    for (int j = 0; j < 2 * T::N; ++j) tiles.load(0, j, 0, true);
#pragma unroll
    for (int j = 0; j < 2 * T::N; ++j)
      if (DEPTH == 2) tiles.load(DEPTH - 1, j, 1, 1 < count);
    tiles.tell(0);
    tiles.turn();
#pragma unroll
    for (int j = 0; j < 2 * T::N; ++j) tiles.store(0, j, k0, v0);
#pragma unroll
    for (int j = 0; j < 2 * T::N; ++j) tiles.load(0, j, DEPTH, DEPTH < count);
  }

  // Tile i of the piece from (kl, vl).  Between the products of the scores the next
  // tile's codes become fp16 in (kn, vn), and the loads of the one after take their
  // registers.  Of a thin row block a wave takes 32 of the keys and half of the channels.
  auto take = [&](int i, auto parity, const uint16_t* kl, const uint16_t* vl, uint16_t* kn, uint16_t* vn) {
    constexpr int SB = THIN ? 1 : ST, DB = THIN ? DT / 2 : DT, VN = DB < 4 ? DB : 4;  // VN: fragments of values read ahead
    const int tb = THIN ? wave & 1 : 0;
    constexpr int next = DEPTH == 1 ? 0 : 1 - decltype(parity)::value;  // the registers of tile i + 1, and of i + 1 + DEPTH
    lds_barrier();
    tiles.step(i);
    const bool more = i + 1 + DEPTH < count;
    auto feed = [&](int j) {
      tiles.store(next, j, kn, vn);
      tiles.load(next, j, i + 1 + DEPTH, more);
    };
    const int place = i % kBatch * 4;
    const int key = (p.t0 + i) * kKeys;
    // the lane's places in the rows; out of the compiler's sight, or it keeps one register
    // for each of their uses.  Row 8 x + 4 h + y of the scores is key 16 h + 4 x + y of
    // its 32: a lane holds 16 keys side by side, of one page.
    const int row_key = 16 * (r >> 2 & 1) + 4 * (r >> 3) + (r & 3);
    int from_k = row_key * D + 8 * (h ^ k_swizzle<D>(row_key)), from_v = r * kKeys + 8 * (2 * h ^ (r >> 1 & 7));
    if (THIN) from_k += 32 * tb * D, from_v = (from_v ^ 32 * tb) + 32 * (wave >> 1) * DB * kKeys;
    asm volatile("" : "+v"(from_k), "+v"(from_v));
    f32x16 s[SB];
#pragma unroll
    for (int t = 0; t < SB; ++t) s[t] = (f32x16)(0.0f);
    constexpr int CH = KK / 4;  // channel steps of a quarter
    f16x8 kf[2][CH][SB];
    auto read_k = [&](int q) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int t = 0; t < SB; ++t) {
          kf[q & 1][k][t] = *reinterpret_cast<const f16x8*>(kl + 32 * t * D + (from_k ^ 16 * (q * CH + k) ^ (q * CH + k >= 8 ? 8 : 0)));
        }
    };
    read_k(0);
    // products before another wave's softmax, those with the values first (2048 on 14336
    // 742 us, and 779 without an order; others took as long or longer)
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q < 3) read_k(q + 1);
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int t = 0; t < SB; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[q & 1][k][t], qf[q * CH + k], s[t], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 2 * T::N; ++j)
        if (j * 4 / (2 * T::N) == q) feed(j);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (D == 256 && !THIN) {  // in vector registers from here, not brought there for each use
#pragma unroll
      for (int t = 0; t < SB; ++t) asm volatile("" : "+v"(s[t]));
    }
    f32x4 say[SB];
#pragma unroll
    for (int t = 0; t < SB; ++t) say[t] = info[i / kBatch & 1][place + 2 * (tb + t) + h];
    const int past = seen - key - 16 * h;  // keys of the lane up to here are seen
    const bool strange = tiles.strange >> place & 1;
    if (__builtin_expect(strange || key + kKeys - 1 > all_see, 0)) {
      const uint32_t held = (uint32_t)(tiles.held >> place) & 15, odd = (uint32_t)(tiles.odd >> place) & 15;
#pragma unroll
      for (int t = 0; t < SB; ++t) {
        if (odd) s[t] *= say[t][0], say[t][0] = 1.0f;
        const int last = held >> (2 * (tb + t) + h) & 1 ? past - 32 * (tb + t) : -1;
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (x > last) s[t][x] = -__builtin_inff();
      }
    }
    f16x8 vf[2][VN], pf[2 * SB];
    auto read_v = [&](int c) {  // group c of fragments: of 16 tokens, or half their channels
#pragma unroll
      for (int d = 0; d < VN; ++d)
        vf[c & 1][d] = *reinterpret_cast<const f16x8*>(vl + 32 * (c * VN % DB + d) * kKeys + (from_v ^ 8 * (c * VN / DB / 2 * 4 + c * VN / DB % 2)));
    };
    float sum;
    auto weigh = [&]() {
      sum = 0.0f;
#pragma unroll
      for (int t = 0; t < SB; ++t) {
        const float lift = say[t][1] + kLift - m;
        float part = 0.0f;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float w = __builtin_amdgcn_exp2f(s[t][x] * say[t][0] + lift);
          part += w;
          pf[2 * t + x / 8][x % 8] = (f16)w;
        }
        sum += part * say[t][2];
      }
    };
    auto highest = [&]() {
      float up = kNoMax;
#pragma unroll
      for (int t = 0; t < SB; ++t) {
        float x = s[t][0];
#pragma unroll
        for (int y = 1; y < 16; ++y) x = __builtin_fmaxf(x, s[t][y]);
        up = __builtin_fmaxf(up, x * say[t][0] + say[t][1]);
      }
      return up;
    };
    auto raise = [&](float up) {
      // row by row: what other rows of the wave see changes no bit of a row
      up = __builtin_fmaxf(up, from_lane(up, lane ^ 32));
      if (!(up > m + kSlack)) up = m;
      const float f = __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= f;
      if constexpr (!THIN) stay_in_accumulators<D>(o);
    };
    if constexpr (!THIN) stay_in_accumulators<D>(o);
    if constexpr (D == 256 && !THIN) {
      // the scores beside their weights do not fit the registers (2048 on 6144 536 us, and
      // 616 with the weights first)
      const float up = highest();
      if (__any(up > m + kSlack)) raise(up);
      weigh();
    } else {
      // with the maximum as it is; a weight that leaves its range shows it to be too low
      weigh();
      f16x8 top = pf[0];
#pragma unroll
      for (int g = 1; g < 2 * SB; ++g) top = __builtin_elementwise_max(top, pf[g]);
      const f16x4 top4 = __builtin_elementwise_max(__builtin_shufflevector(top, top, 0, 1, 2, 3), __builtin_shufflevector(top, top, 4, 5, 6, 7));
      const f16x2 top2 = __builtin_elementwise_max(__builtin_shufflevector(top4, top4, 0, 1), __builtin_shufflevector(top4, top4, 2, 3));
      if (__any(top2[0] > (f16)kMost || top2[1] > (f16)kMost)) {
        raise(highest());
        weigh();
      }
    }
    l += sum;
    read_v(0);
    if (__builtin_expect(strange, 0)) {
      const uint32_t held = (uint32_t)(tiles.held >> place) & 15;
#pragma unroll
      for (int t = 0; t < SB; ++t) {
        const int last = held >> (2 * (tb + t) + h) & 1 ? past - 32 * (tb + t) : -1;
        // a key that is not seen has no weight, and none of a scale that is not finite either
#pragma unroll
        for (int x = 0; x < 16; ++x) pf[2 * t + x / 8][x % 8] = x > last ? (f16)0.0f : pf[2 * t + x / 8][x % 8] * (f16)say[t][3];
      }
    }
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int c = 0; c < 2 * SB * DB / VN; ++c) {
      if (c + 1 < 2 * SB * DB / VN) read_v(c + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < VN; ++d) {
        f32x16& to = o[c * VN % DB + d];
        to = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[c & 1][d], pf[c * VN / DB], to, 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    tiles.step_after(i);
  };
  if (!THIN && wave_row >= rows) {
    // a wave without rows brings the tiles for the others
    auto bring = [&](int i, uint16_t* kn, uint16_t* vn) {
      lds_barrier();
      tiles.step(i);
#pragma unroll
      for (int j = 0; j < 2 * T::N; ++j) {
        tiles.store(0, j, kn, vn);
        tiles.load(0, j, i + 2, i + 2 < count);
      }
      tiles.step_after(i);
    };
    for (int i = 0; i < count; i += 2) {
      bring(i, k1, v1);
      if (i + 1 < count) bring(i + 1, k0, v0);
    }
    // no load is on its way behind this loop, or the compiler waits for it in the other one
    __builtin_amdgcn_s_waitcnt(0);
  } else {
    for (int i = 0; i < count; i += 2) {
      take(i, std::integral_constant<int, 0>(), k0, v0, k1, v1);
      if (i + 1 < count) take(i + 1, std::integral_constant<int, 1>(), k1, v1, k0, v0);
      if constexpr (!THIN) {
        stay_in_accumulators<D>(o);
        if constexpr (D == 256)  // and the queries, so that the codes need not be brought from there
#pragma unroll
          for (int k = 0; k < KK; ++k) asm volatile("" : "+a"(qf[k]));
      }
    }
  }

  l += from_lane(l, lane ^ 32);
  if constexpr (THIN) {
    finish_thin<D>(a, p, kvh, wave, lane, o, m, l, wave < 2 ? k0 : k1, reinterpret_cast<float*>(v0), v1);
  } else {
    finish<D>(a, p, kvh, wave, lane, o, m, l, wave < 2 ? (wave == 0 ? k0 : k1) : (wave == 2 ? v0 : v1));
  }
}

template <int D>
__global__ __launch_bounds__(kWave * kWaves, kPerSimd<D>) void kv8_chunk_kernel(ChunkArgs a) {
  // four arrays and not one: reads of a tile then need not wait for writes of the next
  __shared__ __align__(16) uint16_t k0[kKeys * D], k1[kKeys * D], v0[kKeys * D], v1[kKeys * D];
  __shared__ Info info;
  const int item = a.heads_kv.of(blockIdx.x), kvh = blockIdx.x - item * a.heads_kv.d;
  Piece p;
  {
    const Sizes z = sizes_of(a);
    const Work w = work_of(a, z);
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.slots > 0) *a.plan = w;  // for the join
    if (!piece_of<false>(a, z, w, item, p)) return;
  }
  if (p.block < 0 || p.t0 < 0) return;  // of starts that do not ascend
  if (p.s.n * a.group.d - p.block * kRows <= 32) run<D, true>(a, p, kvh, k0, k1, v0, v1, info);
  else run<D, false>(a, p, kvh, k0, k1, v0, v1, info);
}

// Joins the parts of the row blocks that were cut: 32 rows and 32 channels a
// workgroup, the parts dealt to its waves in turn.
template <int D>
__global__ __launch_bounds__(kWave * kWaves) void kv8_chunk_join_kernel(ChunkArgs a) {
  __shared__ float sm[kWaves][kWave], sl[kWaves][kWave];
  __shared__ f32x4 so[kWaves][4][kWave];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 31, h = lane >> 5;
  constexpr int DT = D / 32;
  const Sizes z = sizes_of(a);
  const Work w = *a.plan;
  for (int x = blockIdx.x;; x += gridDim.x) {
    const int y = a.heads_kv.of(x), kvh = x - y * a.heads_kv.d, d = y % DT, quarter = y / DT % kWaves;
    Piece p;
    if (!piece_of<true>(a, z, w, y / (DT * kWaves), p)) return;
    const int rows = p.s.n * a.group.d, first_row = p.block * kRows + quarter * 32;
    if (first_row >= rows) continue;
    const int row = first_row + r, token = a.group.of(row), q_head = kvh * a.group.d + row - token * a.group.d;
    float m = kNoMax, l = 0.0f;
    f32x4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (f32x4)(0.0f);
    if (row < rows)
      for (int j = wave; j < p.pieces; j += kWaves) {
        const int slot = (p.slot + j) * a.heads_kv.d + kvh;
        if (slot >= a.slots) break;
        const float* part = a.parts + (int64_t)slot * kPartFloats<D>;
        const float pm = part[quarter * 32 + r], pl = part[kRows + quarter * 32 + r];
        const f32x4* from = reinterpret_cast<const f32x4*>(part + 2 * kRows + quarter * 32 * D) + 4 * d * kWave + lane;
        const float up = __builtin_fmaxf(m, pm);
        const float f = __builtin_amdgcn_exp2f(m - up), fp = __builtin_amdgcn_exp2f(pm - up);
        m = up, l = l * f + pl * fp;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * f + from[i * kWave] * fp;
      }
    sm[wave][lane] = m, sl[wave][lane] = l;
#pragma unroll
    for (int i = 0; i < 4; ++i) so[wave][i][lane] = o[i];
    __syncthreads();
    float up = kNoMax, sum = 0.0f;
    f32x4 v = (f32x4)(0.0f);  // wave i: the lane's channels 8 i .. 8 i + 3 past 4 h
#pragma unroll
    for (int j = 0; j < kWaves; ++j) up = __builtin_fmaxf(up, sm[j][lane]);
#pragma unroll
    for (int j = 0; j < kWaves; ++j) {
      const float f = __builtin_amdgcn_exp2f(sm[j][lane] - up);
      sum += sl[j][lane] * f, v += so[j][wave][lane] * f;
    }
    if (row < rows) {
      const float inv = sum > 0.0f ? __builtin_exp2f(-kLift) / sum : sum == 0.0f ? 0.0f : sum;
      u32x2 c;
      c[0] = as_u32((f16x2){(f16)(v[0] * inv), (f16)(v[1] * inv)});
      c[1] = as_u32((f16x2){(f16)(v[2] * inv), (f16)(v[3] * inv)});
      *reinterpret_cast<u32x2*>(a.out + (int64_t)(p.s.first + token) * a.o_token + (int64_t)q_head * a.o_head + 32 * d + 8 * wave + 4 * h) = c;
    }
    __syncthreads();
  }
}

struct Plan {
  int64_t workers, slots, blocks, grid;
  int joined;
  size_t scratch;
};

// Of the lengths that work_of tries, those that cut the longest row block into up to kCuts leave
// each of the others with no more; those that share out what all have in all are at least
// work / workers long, so that the pieces are at most the workers and one for each row block (and
// one, for the share in fp32).  No plan has more parts (24 new tokens, 24 / 4 heads of 256, with a
// table of 32768: 264 of 130 KB, where four for each worker would be 1024).
Plan plan_of(int64_t batch, int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t head_dim, int64_t max_tokens) {
  Plan p;
  p.workers = (head_dim == 64 ? kPerSimd<64> : head_dim == 128 ? kPerSimd<128> : kPerSimd<256>) * (int64_t)lbh::device_cus();
  const int64_t blocks = (tokens * (heads_q / heads_kv) / kRows + batch) * heads_kv;
  const int64_t tiles = (max_tokens + kKeys - 1) / kKeys;
  p.joined = tiles > kMinTiles;
  // no more pieces than all row blocks have of the smallest size
  const int64_t pieces = blocks * ((tiles + kMinTiles - 1) / kMinTiles);
  const int64_t cuts = (kCuts + 1) * blocks, shares = p.workers + blocks + 1;
  p.slots = !p.joined ? 0 : std::min({pieces, kPartRounds * p.workers, std::max(cuts, shares)});
  p.blocks = blocks, p.grid = blocks + p.slots;
  p.scratch = p.slots ? (((size_t)p.slots * kRows * (head_dim + 2) * 4 + 255) & ~(size_t)255) + 256 : 0;
  return p;
}

int check_sizes(int64_t batch, int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t head_dim, int64_t page_size,
                int64_t max_pages) {
  if (batch < 0 || tokens < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0 || max_pages < 0) return LB_ERR_ARG;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LB_ERR_PROB_SHAPE;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return LB_ERR_PROB_SHAPE;
  if (heads_q > 4096 || batch > (1 << 20) || tokens > (1 << 24) || max_pages > (1 << 28) / page_size) return LB_ERR_ARG;
  // tiles and pieces are numbered in 32 bits
  const int64_t blocks = (tokens * (heads_q / heads_kv) / kRows + batch) * heads_kv;
  const int64_t tiles = max_pages * page_size / kKeys + 1;
  if (blocks > (1 << 30) / tiles || tokens * (heads_q / heads_kv) > (1 << 30)) return LB_ERR_PROB_SHAPE;
  return LB_OK;
}

template <int D>
void launch(const ChunkArgs& a, const Plan& p, hipStream_t st) {
  kv8_chunk_kernel<D><<<dim3((unsigned)p.grid), dim3(kWave * kWaves), 0, st>>>(a);
  if (!p.joined) return;
  const int64_t cut = p.blocks < p.workers ? p.blocks : p.workers, units = cut * kWaves * (D / 32), most = 8 * (int64_t)lbh::device_cus();
  kv8_chunk_join_kernel<D><<<dim3((unsigned)(units < most ? units : most)), dim3(kWave * kWaves), 0, st>>>(a);
}

}  // namespace
}  // namespace lb

extern "C" size_t lb_kv8_chunk_attention_scratch_bytes(int64_t batch, int64_t tokens, int64_t heads_q, int64_t heads_kv,
                                                       int64_t head_dim, int64_t page_size, int64_t max_pages) {
  if (lb::check_sizes(batch, tokens, heads_q, heads_kv, head_dim, page_size, max_pages) != LB_OK || batch == 0 || tokens == 0)
    return 0;
  return lb::plan_of(batch, tokens, heads_q, heads_kv, head_dim, page_size * max_pages).scratch;
}

extern "C" int lb_kv8_chunk_attention(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, const int8_t* k_cache,
                                      const int8_t* v_cache, const float* k_scale, const float* v_scale, int64_t num_pages,
                                      int64_t page_size, const int32_t* page_table, int64_t max_pages, int64_t table_stride,
                                      const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t batch, int64_t tokens,
                                      int64_t heads_q, int64_t heads_kv, int64_t head_dim, uint16_t* out,
                                      int64_t o_token_stride, int64_t o_head_stride, float softmax_scale, void* scratch,
                                      size_t scratch_bytes, lb_stream_t stream) {
  using namespace lb;
  const int err = check_sizes(batch, tokens, heads_q, heads_kv, head_dim, page_size, max_pages);
  if (err != LB_OK) return err;
  if (num_pages < 0 || num_pages > 0x7fffffff / heads_kv || table_stride < max_pages) return LB_ERR_ARG;
  if (!(softmax_scale > 0.0f) || softmax_scale > 3e38f) return LB_ERR_ARG;
  if (batch == 0 || tokens == 0) return LB_OK;
  if (!q || !out || !seq_lens || !cu_seqlens) return LB_ERR_ARG;
  if (num_pages > 0 && max_pages > 0 && (!k_cache || !v_cache || !k_scale || !v_scale || !page_table)) return LB_ERR_ARG;
  const void* ptrs[] = {q, out, k_cache, v_cache, scratch};
  for (const void* p : ptrs)
    if (!lbh::aligned(p, 16)) return LB_ERR_ALIGN;
  if ((q_token_stride | q_head_stride | o_token_stride | o_head_stride) % 8 != 0) return LB_ERR_ALIGN;
  // without pages no sequence holds a token
  const int64_t max_tokens = num_pages > 0 ? max_pages * page_size : 0;
  const Plan p = plan_of(batch, tokens, heads_q, heads_kv, head_dim, max_tokens);
  if (p.scratch > 0 && (scratch_bytes < p.scratch || !scratch)) return LB_ERR_SCRATCH;

  ChunkArgs a;
  a.q = q, a.q_token = q_token_stride, a.q_head = q_head_stride;
  a.k_cache = k_cache, a.v_cache = v_cache, a.k_scale = k_scale, a.v_scale = v_scale;
  a.page_table = page_table, a.seq_lens = seq_lens, a.starts = cu_seqlens;
  a.out = out, a.o_token = o_token_stride, a.o_head = o_head_stride;
  a.parts = static_cast<float*>(scratch), a.plan = p.slots ? reinterpret_cast<Work*>(static_cast<char*>(scratch) + p.scratch - 256) : nullptr;
  a.table_stride = table_stride;
  a.num_pages = (int)num_pages, a.page_shift = __builtin_ctzll((unsigned long long)page_size);
  a.max_tokens = (int)max_tokens, a.unit_shift = unit_shift((int)max_tokens);
  a.batch = (int)batch, a.tokens = (int)tokens, a.heads_kv = Divisor((int)heads_kv), a.group = Divisor((int)(heads_q / heads_kv));
  a.workers = (int)p.workers, a.slots = (int)p.slots;
  a.scale = softmax_scale * kLog2e;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (head_dim == 256) launch<256>(a, p, st);
  else if (head_dim == 128) launch<128>(a, p, st);
  else launch<64>(a, p, st);
  return lbh::launch_status();
}
