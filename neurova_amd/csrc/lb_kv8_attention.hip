// Attention of a sequence's newest tokens over its pages of the 8-bit cache.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= len - n + i
//   k[j] = k_scale[page] ck[j],  v[j] = v_scale[page] cv[j]
//
// The cache is read once, so the bound is its bytes: 2 head_dim a token and
// key/value head.  The query heads of a group and the n tokens are the columns
// of both products, 16 or 32 at a time:
//
//   S^T = K Q^T   rows = tokens: the key layout [token][channel] holds a lane's
//                 16 channels of one token together
//   O^T = V^T P^T rows = channels: the value layout [channel][token] gives a
//                 lane 16 tokens of one channel in a 16-byte load
//
// A wave takes 64 tokens a step.  Token 16 g + 4 t + i is row 4 g + i of
// product t, so the accumulators of lane group g are the tokens 16 g .. 16 g + 15
// of its column, in order: exactly the tokens of the lane's value loads.  The
// weights go from the first product to the second without leaving the lane, and
// a lane's tokens share a page (pages hold 16 tokens or more), so both scales
// are one number a lane and step.
//
//   128 sequences of 500 to 8192 tokens, 8 heads of 128: 122 us, 5.5 TB/s where
//   reads alone reach 6.2; one of 131072 tokens, 4 heads of 256: 53 us (5.0 TB/s;
//   49.0 and 4.7 for the join).  Few tokens are bound by the chain of loads that
//   wait for one another (length, page, keys) and a step's instructions, 800 a
//   wave: 301 tokens, 4 heads of 256: 10.6 us, of which 2 are the two loads before
//   the keys, 4 the first step, 1.7 the output.
#include <type_traits>

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
  int workers, cus, min_units, joined;  // joined: a second launch joins the parts
  float scale;  // softmax scale * log2(e)
};

constexpr int kStep = 64;           // tokens a wave takes at a time
constexpr int kStreams = 4;            // streams of tokens in a workgroup
constexpr int kUnit = kStep * kStreams;  // tokens of a unit of work
constexpr float kNoMax = -1e30f;
// The running maximum is that of weight times value scale (a score plus the
// scale's logarithm), which is what the second product takes: a page that a row
// ignores costs the others none of their bits, however large its values.  It moves
// only when exceeded by 2^kSlack, and the weights carry 2^kLift more: at most
// 2^15, inside fp16, and 2^7 farther from its subnormals.  Scales count from
// 2^-kScales to 2^kScales (a page of zeros as the lowest), so that the sums of the
// weights alone stay inside fp32: at most 2^(kSlack + kScales) for each of 2^28
// tokens.
constexpr float kSlack = 8.0f, kLift = 7.0f, kScales = 80.0f;
// Slots may be this many units longer if each then has a compute unit to itself:
// 5 sequences of 700 to 6000 tokens, 3 new ones, 8 heads of 128: 18.0 us with 3
// units in 200 slots, 19.3 with 2 in 280, where the last 24 share theirs.
constexpr int kAlone = 1;
// Above a quarter of the workers, pairs get slots if these are at most this many
// units longer than equal ranges, and so mostly a workgroup each: 64 sequences of
// 300 to 1000 tokens, 8 heads of 64: 15.7 us, with ranges 18.2; of 2000 to 4000
// tokens, 4 heads of 256, where slots of 4 units more would serve: 86.7, 81.8.
constexpr int kWhole = 1;
// A pair's parts are joined by its last worker, or by a second launch with a
// workgroup for each column where pairs that fill their tables have 16 slots or
// more (one sequence, 8 heads of 128: 2500 tokens 10.8 us, with a second launch
// 11.4; 4000 tokens, 16 slots, 12.4 and 10.7; 131072 tokens 182 and 53).  The
// sizes decide, since lengths are on the device: a short sequence in such a table
// pays for the second launch too (301 tokens 8.5 us in a table of 3840, 10.0 in
// one of 4096 or more, 10.9 where each call is launched by itself), which is why it
// does not begin earlier.
constexpr int kManySlots = 16;
constexpr int kParts = 8;        // parts whose loads a thread of the last worker has in flight: 32768
                                 // tokens beside 15 x 300: 30.6 us, 4 at a time 35.8, 16 the same
constexpr int kJoinGroups = 16;  // groups of D / 4 threads that join a column's parts in the second launch

__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + kUnit - 1) / kUnit : 1; }

// Head dimension 256 is two waves of 128 channels for each stream of tokens (the
// registers of all 256 would leave one wave a SIMD; 301 tokens took 14.2 us so,
// 12.5 with the halves): each sums the scores over
// its half, the halves are exchanged through LDS, and both carry the same
// softmax for their half of the output.
template <int D>
constexpr int kHalves = D == 256 ? 2 : 1;
template <int D>
constexpr int kThreads = kWave * kStreams * kHalves<D>;

// Workgroups of a compute unit: two waves a SIMD where the registers allow it.
template <int D, int NQ>
constexpr int kPerCu = D * NQ <= 128 ? 2 : 1;

template <int D, int NQ>
struct Shared {
  static constexpr int kCols = 16 * NQ;
  union {
    float o[kStreams][kCols][D + 4];
    f32x4 s[kHalves<D>][kStreams][kHalves<D>][NQ * 4][kHalves<D> == 2 ? kWave : 1];  // partial scores, two steps of them
  };
  float m[kStreams][kCols], l[kStreams][kCols];
  int last;
};

// How a launch's work is cut.  A pair (sequence, key/value head, column block)
// has `nu` units.  In general the workgroups take equal contiguous ranges of all
// units, numbered pair by pair, so one may end a pair and begin the next.  Where
// the pairs are no more than the workers, each can be cut into slots of its own,
// `per` units or a little less, one a workgroup: the fixed time of a segment (its
// first loads, the join) is then paid once.  Up to a quarter of the workers, pairs
// always are (5 sequences of 700 to 6000 tokens, 3 new ones, 8 heads of 128: 18.6
// us, with ranges 25.6).
struct Work {
  int units, per;
  bool slots;
};

__device__ __forceinline__ int len_at(const AttnArgs& a, int b) {
  return b < a.batch ? max(min(a.seq_lens[b], a.max_tokens), 0) : -1;
}
// Tokens of a sequence past its table: they say which keys the new ones see.
__device__ __forceinline__ int past_at(const AttnArgs& a, int b) {
  return b < a.batch ? max(a.seq_lens[b], a.max_tokens) - a.max_tokens : 0;
}
// Units of a sequence's pairs; 0 past the batch (length -1).
__device__ __forceinline__ int units_or_none(int len) { return len < 0 ? 0 : units_of(len); }

// Slots of a pair: ceil(nu / per), for nu <= 2^20 and per <= nu or so.  A float
// product is exact enough: (x + 1/2) / per is 1 / (2 per) away from an integer,
// more than its error of x / per * 2^-22.
__device__ __forceinline__ int slots_in(int nu, int per, float inverse) {
  return (int)(((float)(nu + per - 1) + 0.5f) * inverse);
}

// The smallest slots from `per` to `last` units of which there are at most
// `most`; 0 if there are none.
__device__ __forceinline__ int slots_for(const AttnArgs& a, int first_len, int per, int last, int most) {
  const int per_seq = a.heads_kv * a.col_blocks;
  for (; per <= last; ++per) {
    const float inverse = __builtin_amdgcn_rcpf((float)per);
    int slots = 0;
    for (int c = 0; c < a.batch; c += kWave)
      slots += __builtin_amdgcn_readlane(
          wave_scan(slots_in(units_or_none(c ? len_at(a, c + lane_id()) : first_len), per, inverse)), kWave - 1);
    if (slots * per_seq <= most) return per;
  }
  return 0;
}

__device__ __forceinline__ Work work_of(const AttnArgs& a, int first_len) {
  int total = __builtin_amdgcn_readlane(wave_scan(units_or_none(first_len)), kWave - 1);
  for (int c = kWave; c < a.batch; c += kWave)
    total += __builtin_amdgcn_readlane(wave_scan(units_or_none(len_at(a, c + lane_id()))), kWave - 1);
  const int per_seq = a.heads_kv * a.col_blocks, pairs = a.batch * per_seq;
  Work w;
  w.units = total * per_seq;
  w.per = max((w.units + a.workers - 1) / a.workers, a.min_units);
  w.slots = false;
  if (pairs <= a.workers) {
    int per = 0;
    const int alone = max((w.units + a.cus - 1) / a.cus, a.min_units);
    if (a.workers > a.cus) per = slots_for(a, first_len, alone, w.per + kAlone, a.cus);
    // at the latest units / (workers - pairs): there are at most units / per + pairs
    if (!per) per = slots_for(a, first_len, w.per, 4 * pairs <= a.workers ? max(w.units, w.per) : w.per + kWhole, a.workers);
    if (per) w.slots = true, w.per = per;
  }
  return w;
}

// One (sequence, key/value head, column block) over units [u0, u1) of its nu.
struct Segment {
  int b, head, cb, u0, u1, nu, len;
  int w_first, w_last;  // the workers of the whole pair
  int pair;
  int past;  // tokens past the table; in a vector register, the scalar ones are all taken
};

// Four channels of an output row, divided by the sum of the weights (a row that
// saw no key is zero).
__device__ __forceinline__ void store_out(const AttnArgs& a, int b, int head, int col, int d, f32x4 x, float sum) {
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
  const int i = col / a.group;
  uint16_t* row = a.out + ((int64_t)b * a.new_tokens + i) * a.o_token +
                  (int64_t)(head * a.group + (col - i * a.group)) * a.o_head + d;
  u32x2 w;
  w[0] = as_u32((f16x2){(f16)(x[0] * inv), (f16)(x[1] * inv)});
  w[1] = as_u32((f16x2){(f16)(x[2] * inv), (f16)(x[3] * inv)});
  *reinterpret_cast<u32x2*>(row) = w;
}

// A part: the columns' maxima, their sums, then o [column][channel].
template <int D, int NQ>
constexpr int kPartFloats = 16 * NQ * (D + 2);

// Worker w's part of a pair that begins with worker w_first: its first if the
// pair began before it, else its second (a pair that ends after it).
template <int D, int NQ>
__device__ __forceinline__ int64_t part_at(int w, int w_first) {
  return ((int64_t)w * 2 + (w > w_first ? 0 : 1)) * kPartFloats<D, NQ>;
}

// The segments of a worker, in order.
struct Segments {
  Work work;
  int worker, pairs;  // pairs of a sequence
  int u, u_end;       // position: in units, or with slots in slots
  int chunk, at, base;  // sequence chunk + at, which begins at position base
  int lens, past;       // lengths of the 64 sequences from chunk on, and what the table leaves out of them

  __device__ __forceinline__ bool begin(const AttnArgs& a) {
    const int lane = lane_id();
    pairs = a.heads_kv * a.col_blocks;
    lens = len_at(a, lane), past = past_at(a, lane);
    work = work_of(a, lens);
    worker = blockIdx.x;
    u = work.slots ? worker : worker * work.per;
    u_end = 0, chunk = 0, base = 0;
    int size, upto;
    for (;;) {
      const int nu = units_or_none(lens);
      size = (work.slots ? (nu + work.per - 1) / work.per : nu) * pairs;
      upto = wave_scan(size);
      const int all = __builtin_amdgcn_readlane(upto, kWave - 1);
      if (base + all > u) break;
      base += all, chunk += kWave;
      if (chunk >= a.batch) return false;
      lens = len_at(a, chunk + lane), past = past_at(a, chunk + lane);
    }
    at = __builtin_ctzll(__ballot(base + upto > u));  // the sequence that holds u
    base += __builtin_amdgcn_readlane(upto - size, at);
    u_end = work.slots ? u + 1 : min(work.units, u + work.per);
    return true;
  }

  __device__ __forceinline__ bool next(const AttnArgs& a, Segment& sg) {
    if (u >= u_end) return false;
    const int len = __builtin_amdgcn_readlane(lens, at), nu = units_of(len);
    const int slots = work.slots ? (nu + work.per - 1) / work.per : nu;
    const int x = (u - base) / slots, first = base + x * slots;
    sg.b = chunk + at, sg.nu = nu, sg.len = len;
    sg.head = x / a.col_blocks, sg.cb = x - sg.head * a.col_blocks;
    sg.pair = sg.b * pairs + x;
    sg.past = (int)from_lane((uint32_t)past, at);
    if (work.slots) {
      const int i = u - first;
      sg.u0 = nu * i / slots, sg.u1 = nu * (i + 1) / slots;  // nu <= 2^20, slots <= workers
      sg.w_first = first, sg.w_last = first + slots - 1;
      u = u_end;
    } else {
      sg.u0 = u - first, sg.u1 = min(nu, u_end - first);
      sg.w_first = first / work.per, sg.w_last = (first + nu - 1) / work.per;
      u = first + sg.u1;
      if (u < u_end && x == pairs - 1 && sg.u1 == nu) {  // on to the next sequence
        base += nu * pairs;
        if (++at == kWave) at = 0, chunk += kWave, lens = len_at(a, chunk + lane_id()), past = past_at(a, chunk + lane_id());
      }
    }
    return true;
  }
};

// A wave's walk over the steps of its worker's segments, with the loads of one
// step ahead: the registers that a product has read are loaded for the next
// step at once, also across the end of a segment, so that its join runs while
// the next segment's first keys and values are on their way.  ONCE: the pair has
// one column block, so its keys and values are read once and need no place in
// the caches (64 sequences of 2000 to 4000 tokens, 8 heads of 128: 84 us against
// 77; with two column blocks the second one's reads would miss: 27 against 30).
template <int D, int NQ, bool ONCE>
struct Walk {
  static constexpr int H = kHalves<D>, DW = D / H, KI = DW / 64, VT = DW / 16, COLS = 16 * NQ;
  const AttnArgs& a;
  Shared<D, NQ>& sh;
  int lane, r, g, stream, half;
  // the step whose keys and values are loaded, or on their way
  const int8_t* vp;
  int cell;  // page and head of the lane's own 16 tokens
  float ks, vs;
  bool held;
  u32x4 vw[VT];
  uint8_t* keys;        // this wave's keys of a step in LDS
  uint32_t k_off[4];    // the lane's place in a load of 16-token group i
  const int8_t* k_base[4];  // where the groups' keys are
  int pv;               // page number of the lane's own 16 tokens in the step after
  bool loaded, pages_known;
  f16x8 qf[NQ][2 * KI];
  int limit[NQ];  // keys that the lane's columns see
  int flip;       // which of the two score buffers

  __device__ __forceinline__ Walk(const AttnArgs& args, Shared<D, NQ>& shared, uint8_t* lds) : a(args), sh(shared) {
    lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    stream = wave % kStreams, half = H == 1 ? 0 : wave / kStreams;
    loaded = pages_known = false, flip = 0, pv = -1;
    keys = lds + wave * kStep * DW;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      k_off[i] = DW == 64 ? (lane >> 2) * D + ((lane & 3) ^ i) * 16
                          : (lane >> 3) * D + ((lane & 7) ^ (2 * i + ((lane >> 4) & 1))) * 16;
  }
  __device__ __forceinline__ int first_token(const Segment& sg) const { return sg.u0 * kUnit + stream * kStep; }
  __device__ __forceinline__ static int end_token(const Segment& sg) { return min(sg.len, sg.u1 * kUnit); }

  // Page numbers of the step of sequence b at token tb.  No branch around the
  // load (a token past the end reads the last one's): the waits inside the loop
  // over the steps count the loads between.
  __device__ __forceinline__ void fetch_pages(int b, int len, int tb) {
    pv = a.page_table[(int64_t)b * a.table_stride + (min(tb + 16 * g, len - 1) >> a.page_shift)];
  }
  __device__ __forceinline__ void resolve(const Segment& sg, int tb) {
    const int tv = tb + 16 * g, mask = (1 << a.page_shift) - 1;
    held = tv < sg.len && (unsigned)pv < (unsigned)a.num_pages;
    const int page = held ? pv : 0;
    cell = page * a.heads_kv + sg.head;
    const int64_t cv = cell;
    vp = a.v_cache + ((cv * D + half * DW + r) << a.page_shift) + (tv & mask);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t ck = (int64_t)__builtin_amdgcn_readlane(page, 16 * i) * a.heads_kv + sg.head;
      k_base[i] = a.k_cache + ((ck << a.page_shift) + ((tb + 16 * i) & mask)) * D + half * DW;
    }
  }
  __device__ __forceinline__ void load_scales() { ks = a.k_scale[cell], vs = a.v_scale[cell]; }
  // Keys of a step go through LDS: a load of 1 KB takes whole cache lines, which
  // the first product's operand (one token a lane) would touch one lane at a
  // time, a quarter of the first-level cache's rate.  Chunks of 16 bytes change
  // places inside a row so that the reads of a product's 16 tokens use every bank.
  __device__ __forceinline__ void load_k() {
    typedef __attribute__((address_space(3))) void lds_void;
    constexpr int N = DW / 64;  // loads of a group of 16 tokens
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
      const __amdgpu_buffer_rsrc_t from = buffer_of(k_base[i / N], 16 * D - half * DW);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)(keys + i * 1024), 16, k_off[i / N], (i % N) * 8 * D, 0, ONCE ? kNonTemporal : 0);
    }
  }
  __device__ __forceinline__ u32x4 read_k(int t, int i) const {
    const int token = 16 * (r >> 2) + 4 * t + (r & 3), chunk = g + 4 * i;
    const int swz = DW == 64 ? token >> 4 : 2 * (token >> 4) + ((token >> 1) & 1);
    return *reinterpret_cast<const u32x4*>(keys + token * DW + (chunk ^ swz) * 16);
  }
  __device__ __forceinline__ void load_v(int d) {
    const u32x4* from = reinterpret_cast<const u32x4*>(vp + ((int64_t)(16 * d) << a.page_shift));
    vw[d] = ONCE ? __builtin_nontemporal_load(from) : *from;
  }
  // The query fragments, in the channel order of the key loads.
  __device__ __forceinline__ void load_q(const Segment& sg) {
    const int cols = a.new_tokens * a.group;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int col = sg.cb * COLS + 16 * n + r;
      const int i = col / a.group;
      limit[n] = col < cols ? sg.len - a.new_tokens + i + 1 + sg.past : 0;
      const uint16_t* row = a.q + ((int64_t)sg.b * a.new_tokens + i) * a.q_token +
                            (int64_t)(sg.head * a.group + (col - i * a.group)) * a.q_head + half * DW + 16 * g;
#pragma unroll
      for (int k = 0; k < 2 * KI; ++k) {
        qf[n][k] = (f16x8)((f16)0.0f);
        if (col < cols) qf[n][k] = *reinterpret_cast<const f16x8*>(row + 64 * (k / 2) + 8 * (k & 1));
      }
    }
  }
  __device__ __forceinline__ static int steps_from(int tb, int end) { return tb < end ? (end - tb + kUnit - 1) / kUnit : 0; }
  // The pages of the step after the next one, at token tp of sg or past its end,
  // where that is known by now: in `to`, if it follows.
  __device__ __forceinline__ void fetch_after(const Segment& sg, int tp, bool ahead, const Segment& to) {
    const bool inside = tp < end_token(sg);
    const bool beyond = !inside && ahead && first_token(to) < end_token(to);
    pages_known = inside || beyond;
    fetch_pages(beyond ? to.b : sg.b, beyond ? to.len : sg.len, inside ? tp : beyond ? first_token(to) : 0);
  }
  // Loads of a step that nothing was loaded ahead of.
  __device__ __forceinline__ void start(const Segment& sg, bool ahead, const Segment& to) {
    const int tb = first_token(sg);
    if (loaded || tb >= end_token(sg)) return;
    if (!pages_known) fetch_pages(sg.b, sg.len, tb);
    resolve(sg, tb);
    fetch_after(sg, tb + kUnit, ahead, to);
    load_k();
    __builtin_amdgcn_sched_barrier(0);  // the values' loads after the keys'
    load_scales();
#pragma unroll
    for (int d = 0; d < VT; ++d) load_v(d);
    __builtin_amdgcn_sched_barrier(0);
    loaded = true;
  }

  // One step of segment sg at token tb: the last of the segment or (LAST false)
  // not; with MORE another one follows, in sg or in `to`.
  template <bool MORE, bool LAST>
  __device__ __forceinline__ void step(const Segment& sg, int tb, f32x4 (&o)[NQ][VT], float (&m)[NQ], float (&l)[NQ],
                                       bool ahead, const Segment& to) {
    const bool held0 = held;
    // the keys are in LDS once no more loads are out than those of the values,
    // which follow theirs (nothing else waits for a load into LDS here)
    static_assert(VT < 16, "the low bits of the counter");
    __builtin_amdgcn_s_waitcnt(0x0f70 | VT);  // vmcnt(VT)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    u32x4 kw[4][KI];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < KI; ++i) kw[t][i] = read_k(t, i);
    if (MORE) {
      if (LAST) {
        if (!pages_known) fetch_pages(to.b, to.len, first_token(to));
        resolve(to, first_token(to));
        fetch_after(to, first_token(to) + kUnit, false, to);
      } else {
        resolve(sg, tb + kUnit);
        fetch_after(sg, tb + 2 * kUnit, ahead, to);
      }
      // the reads above are done: the next keys may take their place
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      load_k();
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x4 s[NQ][4];
    // two products at a time, each in two sums: four independent chains of MFMAs
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      f32x4 odd[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][t] = s[n][t + 1] = odd[n][0] = odd[n][1] = (f32x4)(0.0f);
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f16x8 x, y;
          codes_to_half(kw[t + u][i], x, y);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            s[n][t + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qf[n][2 * i], s[n][t + u], 0, 0, 0);
            odd[n][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, qf[n][2 * i + 1], odd[n][u], 0, 0, 0);
          }
        }
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][t] += odd[n][0], s[n][t + 1] += odd[n][1];
    }
    if (H == 2) {
      // a step's buffer is written again two steps later, behind the barrier
      // that the partner reaches after its reads
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int t = 0; t < 4; ++t) sh.s[flip][stream][half][4 * n + t][lane] = s[n][t];
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[n][t] += sh.s[flip][stream][half ^ 1][4 * n + t][lane];
      flip ^= 1;
    }
    const int tv = tb + 16 * g;
    // a scale of infinity has no scores (those below zero would have no weight and
    // its keys go unseen): ks - ks makes it NaN and is zero otherwise
    const float kscale = held0 ? ks * a.scale + (ks - ks) : 0.0f;
    const float vlog = __builtin_fmaxf(__builtin_fminf(__builtin_amdgcn_logf(__builtin_fabsf(vs)), kScales), -kScales);
    const bool mask = tb + kStep > sg.len - a.new_tokens + 1 || __any(!held0);
    float peak[NQ];
    bool up = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      peak[n] = kNoMax;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[n][t][i] * kscale;
          if (mask && (!held0 || tv + 4 * t + i >= limit[n])) x = -__builtin_inff();
          s[n][t][i] = x;
          peak[n] = __builtin_fmaxf(peak[n], x);
        }
      peak[n] += vlog;
      up |= peak[n] > m[n] + kSlack;
    }
    if (__any(up)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float x = __builtin_fmaxf(peak[n], m[n]);
        x = __builtin_fmaxf(x, from_lane(x, lane ^ 16));
        x = __builtin_fmaxf(x, from_lane(x, lane ^ 32));
        const float f = __builtin_amdgcn_exp2f(m[n] - x);
        m[n] = x;
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < VT; ++d) o[n][d] *= f;
      }
    }
    // the weights p * v_scale enter the second product relative to the largest
    // of them, as the sum of two fp16 numbers (one alone would add as much error
    // as the rounding of the output; the matrix cores are mostly idle here).  Both
    // are cut off towards zero by an instruction that takes no part in a fused
    // one: the first has to be the same number in the product and in the rest.
    // A column that sees none of a lane's tokens takes zero for their scale: its
    // weights are zero, and zero times a scale that is not finite is not.
    const float lifted = vs * __builtin_exp2f(kLift);
    f16x8 pf[NQ][2], pl[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float vscale = held0 && tv < limit[n] ? lifted : 0.0f;
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[n][2 * f + j / 4][j % 4 + i] - m[n]);
            l[n] += p;
            w[i] = p * vscale;
          }
          const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(w[0], w[1]));
          const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(w[0] - (float)hi[0], w[1] - (float)hi[1]));
#pragma unroll
          for (int i = 0; i < 2; ++i) pf[n][f][j + i] = hi[i], pl[n][f][j + i] = lo[i];
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (MORE) load_scales();
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
      if (MORE) load_v(d);
      if ((d & 3) == 3) __builtin_amdgcn_sched_barrier(0);
    }
    loaded = MORE;
  }

  // All steps of segment sg, and its join; `ahead`: segment `to` follows.
  __device__ __forceinline__ void run(const Segment& sg, bool ahead, const Segment& to, int worker) {
    f32x4 o[NQ][VT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = kNoMax, l[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < VT; ++d) o[n][d] = (f32x4)(0.0f);
    }
    start(sg, ahead, to);
    const int end = end_token(sg);
    int tb = first_token(sg);
    for (; tb + kUnit < end; tb += kUnit) step<true, false>(sg, tb, o, m, l, ahead, to);
    if (tb < end) {
      if (ahead && first_token(to) < end_token(to)) step<true, true>(sg, tb, o, m, l, ahead, to);
      else step<false, true>(sg, tb, o, m, l, ahead, to);
    }
    // a round of steps in which this stream has none: its barrier all the same
    if (H == 2 && end > sg.u0 * kUnit && steps_from(first_token(sg), end) < steps_from(sg.u0 * kUnit, end)) lds_barrier();
    if (ahead) load_q(to);

    // the streams' states -> one
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      l[n] += from_lane(l[n], lane ^ 16);
      l[n] += from_lane(l[n], lane ^ 32);
      if (g == 0 && half == 0) sh.m[stream][16 * n + r] = m[n], sh.l[stream][16 * n + r] = l[n];
    }
    lds_barrier();
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int c = 16 * n + r;
      float up = kNoMax;
#pragma unroll
      for (int w = 0; w < kStreams; ++w) up = __builtin_fmaxf(up, sh.m[w][c]);
      const float f = __builtin_amdgcn_exp2f(m[n] - up - kLift);
#pragma unroll
      for (int d = 0; d < VT; ++d)
        *reinterpret_cast<f32x4*>(&sh.o[stream][c][half * DW + 16 * d + 4 * g]) = o[n][d] * f;
    }
    lds_barrier();

    const bool whole = sg.u0 == 0 && sg.u1 == sg.nu;
    const int cols = a.new_tokens * a.group;
    const int live = min(COLS, cols - sg.cb * COLS);  // columns of this block that exist
    float* part = a.parts + part_at<D, NQ>(worker, sg.w_first);
    const __amdgpu_buffer_rsrc_t dst = buffer_of(part, kPartFloats<D, NQ> * 4);
    for (int x = threadIdx.x; x < live * (D / 4); x += kThreads<D>) {
      const int c = x / (D / 4), d = 4 * (x % (D / 4));
      float up = kNoMax, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kStreams; ++w) up = __builtin_fmaxf(up, sh.m[w][c]);
#pragma unroll
      for (int w = 0; w < kStreams; ++w) sum += sh.l[w][c] * __builtin_amdgcn_exp2f(sh.m[w][c] - up);
      f32x4 v = (f32x4)(0.0f);
#pragma unroll
      for (int w = 0; w < kStreams; ++w) v += *reinterpret_cast<const f32x4*>(&sh.o[w][c][d]);
      if (whole) {
        store_out(a, sg.b, sg.head, sg.cb * COLS + c, d, v, sum);
      } else {
        if (d == 0) publish(part + c, up), publish(part + COLS + c, sum);
        publish16(dst, (2 * COLS + c * D + d) * 4, v);
      }
    }
    if (whole || a.joined) {
      lds_barrier();  // the next segment writes the shared states again
      return;
    }
    // the last of the pair's workers to arrive joins the parts, in worker order
    wait_published();
    __syncthreads();
    if (threadIdx.x == 0) sh.last = arrive(a.counters + sg.pair) == sg.w_last - sg.w_first;
    __syncthreads();
    if (sh.last) join(sg, live);
    __syncthreads();
  }

  __device__ __forceinline__ void join(const Segment& sg, int live) {
    after_last_arrival();
    for (int x = threadIdx.x; x < live * (D / 4); x += kThreads<D>) {
      const int c = x / (D / 4), d = 4 * (x % (D / 4));
      float up = kNoMax, sum = 0.0f;
      f32x4 v = (f32x4)(0.0f);
      for (int w0 = sg.w_first; w0 <= sg.w_last; w0 += kParts) {
        float pm[kParts], pl[kParts];
        f32x4 po[kParts];
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          pm[i] = kNoMax, pl[i] = 0.0f, po[i] = (f32x4)(0.0f);
          if (w0 + i <= sg.w_last) {
            const __amdgpu_buffer_rsrc_t from =
                buffer_of(a.parts + part_at<D, NQ>(w0 + i, sg.w_first), kPartFloats<D, NQ> * 4);
            pm[i] = collect4(from, c * 4);
            pl[i] = collect4(from, (COLS + c) * 4);
            po[i] = collect16(from, (2 * COLS + c * D + d) * 4);
          }
        }
        float top = up;
#pragma unroll
        for (int i = 0; i < kParts; ++i) top = __builtin_fmaxf(top, pm[i]);
        const float f0 = __builtin_amdgcn_exp2f(up - top);
        up = top, sum *= f0, v *= f0;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          const float f = __builtin_amdgcn_exp2f(pm[i] - top);
          sum += pl[i] * f, v += po[i] * f;
        }
      }
      store_out(a, sg.b, sg.head, sg.cb * COLS + c, d, v, sum);
    }
    if (threadIdx.x == 0) reset_counter(a.counters + sg.pair);
  }
};

template <int D, int NQ, bool ONCE>
__global__ __launch_bounds__(kThreads<D>, (kPerCu<D, NQ>)) void kv8_attention_kernel(AttnArgs a) {
  __shared__ Shared<D, NQ> sh;
  __shared__ __align__(16) uint8_t keys[kStreams * kStep * D];
  Segments segments;
  if (!segments.begin(a)) return;
  Segment cur, to;
  bool have = segments.next(a, cur);
  Walk<D, NQ, ONCE> walk(a, sh, keys);
  if (have) {
    walk.start(cur, false, cur);
    walk.load_q(cur);
  }
  while (have) {
    have = segments.next(a, to);
    walk.run(cur, have, to, segments.worker);
    cur = to;
  }
}

// Joins the parts of the pairs that several workers share, one column of one
// pair a workgroup: D / 4 threads a part, the parts dealt to the thread groups
// in turn and their sums added in group order.  With this launch the pairs are at
// most a sixteenth of the workers (kManySlots), 32 on 256 compute units: their
// sequences' lengths fit a wave, and they are cut into slots.
template <int D, int NQ>
__global__ __launch_bounds__(kJoinGroups * D / 4) void kv8_join_kernel(AttnArgs a) {
  constexpr int COLS = 16 * NQ, T = D / 4, GROUPS = kJoinGroups;
  __shared__ float sm[GROUPS], sl[GROUPS];
  __shared__ f32x4 so[GROUPS][T];
  const int pairs = a.heads_kv * a.col_blocks;
  const int c = blockIdx.x % COLS, pair = blockIdx.x / COLS;
  const int b = pair / pairs, x = pair % pairs, cb = x % a.col_blocks, head = x / a.col_blocks;
  if (cb * COLS + c >= a.new_tokens * a.group) return;
  const int lens = len_at(a, lane_id()), per = work_of(a, lens).per;
  const int size = (units_or_none(lens) + per - 1) / per, upto = wave_scan(size);
  const int slots = __builtin_amdgcn_readlane(size, b);
  const int w_first = __builtin_amdgcn_readlane(upto - size, b) * pairs + x * slots, w_last = w_first + slots - 1;
  if (slots == 1) return;  // one worker held the whole pair and stored its rows
  const int grp = threadIdx.x / T, d = 4 * (threadIdx.x % T);
  float m = kNoMax, l = 0.0f;
  f32x4 o = (f32x4)(0.0f);
#pragma unroll 4
  for (int w = w_first + grp; w <= w_last; w += GROUPS) {
    const float* p = a.parts + part_at<D, NQ>(w, w_first);
    const float pm = p[c], pl = p[COLS + c];
    const f32x4 po = *reinterpret_cast<const f32x4*>(p + 2 * COLS + c * D + d);
    const float up = __builtin_fmaxf(m, pm);
    const float f = __builtin_amdgcn_exp2f(m - up), fp = __builtin_amdgcn_exp2f(pm - up);
    m = up, l = l * f + pl * fp, o = o * f + po * fp;
  }
  if (d == 0) sm[grp] = m, sl[grp] = l;
  so[grp][threadIdx.x % T] = o;
  __syncthreads();
  if (grp != 0) return;
  float up = kNoMax, sum = 0.0f;
  f32x4 v = (f32x4)(0.0f);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) up = __builtin_fmaxf(up, sm[i]);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const float f = __builtin_amdgcn_exp2f(sm[i] - up);
    sum += sl[i] * f, v += so[i][threadIdx.x] * f;
  }
  store_out(a, b, head, cb * COLS + c, d, v, sum);
}

struct Plan {
  int nq, col_blocks, min_units, joined;
  int64_t workers, counters;
  size_t scratch;
};

// A worker for each workgroup that the compute units hold at once; fewer where the
// longest possible sequences hold fewer units.  Up to 16 columns (query heads of
// a group times new tokens) are one column group, above that two at a time share
// a key or value's conversion, but for 256 channels, where they do not fit the
// registers.  The smallest slot is one unit for one column group and two for two,
// whose parts take twice the work to join (1000 tokens, 8 heads of 128, one new:
// 9.5 us, with two units 11.2; four new, 20 columns, 3000 tokens: 20.6, with two
// units 19.0).
Plan plan_of(int64_t batch, int64_t new_tokens, int64_t heads_q, int64_t heads_kv, int64_t head_dim,
             int64_t max_tokens) {
  Plan p;
  const int64_t cols = new_tokens * (heads_q / heads_kv);
  p.nq = cols > 16 && head_dim < 256 ? 2 : 1;
  p.col_blocks = (int)((cols + 16 * p.nq - 1) / (16 * p.nq));
  const int64_t units = max_tokens > 0 ? (max_tokens + kUnit - 1) / kUnit : 1;
  p.counters = batch * heads_kv * p.col_blocks;
  const int64_t most = (head_dim * p.nq <= 128 ? 2 : 1) * (int64_t)lbh::device_cus();
  p.workers = p.counters * units < most ? p.counters * units : most;
  if (4 * p.counters > p.workers && p.workers < most) p.workers = 4 * p.counters < most ? 4 * p.counters : most;
  // parts of a pair where all sequences fill the table (with one long sequence
  // among short ones it may have more; the last worker then joins those too)
  const int64_t per = (p.counters * units + p.workers - 1) / p.workers;
  p.min_units = p.nq;
  p.joined = units / (per > p.min_units ? per : p.min_units) >= kManySlots;
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

template <int D, int NQ>
void launch(const AttnArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.workers), block(kThreads<D>);
  // 64 and 128 channels: up to 16 columns are always one block
  if (p.col_blocks == 1) kv8_attention_kernel<D, NQ, true><<<grid, block, 0, st>>>(a);
  else if constexpr (D == 256 || NQ == 2) kv8_attention_kernel<D, NQ, false><<<grid, block, 0, st>>>(a);
  if (p.joined) kv8_join_kernel<D, NQ><<<dim3((unsigned)(p.counters * 16 * NQ)), dim3(kJoinGroups * D / 4), 0, st>>>(a);
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

extern "C" int lb_kv8_attention_describe_plan(int64_t batch, int64_t tokens, int64_t heads_q, int64_t heads_kv,
                                              int64_t head_dim, int64_t page_size, int64_t max_pages, int64_t* out) {
  if (!out) return LB_ERR_ARG;
  const int err = lb::check_sizes(batch, tokens, heads_q, heads_kv, head_dim, page_size, max_pages);
  if (err != LB_OK) return err;
  for (int i = 0; i < 7; ++i) out[i] = 0;
  if (batch == 0 || tokens == 0) return LB_OK;
  const lb::Plan p = lb::plan_of(batch, tokens / batch, heads_q, heads_kv, head_dim, page_size * max_pages);
  out[0] = 16 * p.nq, out[1] = p.col_blocks, out[2] = p.workers, out[3] = p.min_units * lb::kUnit;
  out[4] = 1 + p.joined, out[5] = p.counters, out[6] = (int64_t)p.scratch;
  return LB_OK;
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
  if (num_pages < 0 || num_pages > 0x7fffffff / heads_kv || table_stride < max_pages) return LB_ERR_ARG;
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
  a.workers = (int)p.workers, a.cus = lbh::device_cus(), a.min_units = p.min_units, a.joined = p.joined;
  a.scale = softmax_scale * kLog2e;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (head_dim == 256) launch<256, 1>(a, p, st);
  else if (head_dim == 128) p.nq == 1 ? launch<128, 1>(a, p, st) : launch<128, 2>(a, p, st);
  else p.nq == 1 ? launch<64, 1>(a, p, st) : launch<64, 2>(a, p, st);
  return lbh::launch_status();
}
