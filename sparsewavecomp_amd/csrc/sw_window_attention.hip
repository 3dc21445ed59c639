// Attention over a sliding window with sinks, forward and backward, for packed
// sequences on gfx950.
//
// Query i of a sequence of nq queries and nk keys stands at p = i + nk - nq
// and sees key j where j <= p and (p - j < window or j < sinks):
//   s = alpha q.k,  m = max s,  l = sum exp(s - m),
//   o = sum exp(s - m) v / l,  log_sum = m + log l.
// Query heads g G .. g G + G - 1 share key head g, G = query_heads / key_heads.
// With p = exp(s - log_sum) and the output's gradient do:
//   dv = sum p do,  dp = do.v,  delta = do.o,  ds = p (dp - delta),
//   dq = alpha sum ds k,  dk = alpha sum ds q,
// the sums for keys over all queries that see them, of all heads that share
// the key head.  The scores are computed again, once for dq and once for dk
// and dv, so that every sum has one owner: no atomics, the same bits again.
#include "sw_heads.h"
#include "sw_internal.h"

#include <algorithm>
#include <cmath>

using namespace swd;
using sw::Operand;
using sw::check_operand;
using sw::operand;

namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kInf = __builtin_inff();

constexpr int kThreads = 256; // four waves, of 32 rows each
constexpr int kRowShift = 7;
constexpr int kRows = 1 << kRowShift;

// The rows of a workgroup whose four waves take their keys in one share, 128,
// or in two, 64 where there are few rows.
constexpr int shared_shift(int streams) { return kRowShift + 1 - streams; }

struct WindowArgs {
  const int32_t *query_offsets, *key_offsets;
  const void *query, *key, *value;
  void *output;
  float *log_sum;
  Operand q, k, v, o;
  int sequences, query_tokens, key_tokens, query_heads, key_heads, d;
  int window, sinks;
  float alpha;
  int tiles; // row tiles of all sequences
};

// One sequence's tokens, within the operands whatever the offsets hold.
struct Sequence {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ int clamped(int x, int lo, int hi) {
  return x < lo ? lo : x > hi ? hi : x;
}
template <typename A>
__device__ __forceinline__ Sequence sequence(const A &a, int i) {
  Sequence s;
  s.q0 = clamped(a.query_offsets[i], 0, a.query_tokens);
  s.nq = clamped(a.query_offsets[i + 1], s.q0, a.query_tokens) - s.q0;
  s.k0 = clamped(a.key_offsets[i], 0, a.key_tokens);
  s.nk = clamped(a.key_offsets[i + 1], s.k0, a.key_tokens) - s.k0;
  return s;
}

// A workgroup's rows: 1 << SHIFT queries of one head, 32 a wave.  Neighbouring
// workgroups of an XCD take the heads that share a key head, then the next
// rows, whose windows overlap (65,536 queries, window 4096: 2222 us; in plain
// order 2351 us).
template <int SHIFT> struct Rows {
  Sequence s;
  int head, key_head, row0, row_lo, count, shift;
  __device__ __forceinline__ Rows(const WindowArgs &a, int block) {
    const int group = a.query_heads / a.key_heads;
    int64_t item = xcd_contiguous(blockIdx.x, gridDim.x);
    const int g = (int)(item % group);
    item /= group;
    const int tile = (int)(item % a.tiles);
    key_head = (int)(item / a.tiles);
    head = key_head * group + g;
    const int i =
        sequence_of_tile(a.query_offsets, a.sequences, tile, SHIFT);
    s = sequence(a, i);
    row0 = (tile - (a.query_offsets[i] >> SHIFT) - i) << SHIFT;
    // (none in the numbers between one sequence's tiles and the next's)
    const int left = s.nq - row0;
    count = row0 < 0 ? 0 : left < 1 << SHIFT ? left : 1 << SHIFT;
    row_lo = row0 + 32 * block;
    shift = s.nk - s.nq; // a query's place less its index
  }
};

// The keys that a workgroup's rows see between them, as tiles of KT: the sinks
// before the window first where they do not touch it, then the window from its
// first key on.  A tile holds keys from .. end - 1; `sink` ones are seen by
// every row.
template <int KT> struct KeyTiles {
  int sink_end, lo, hi, sink_tiles, count;
  __device__ __forceinline__ KeyTiles(int first, int last, int window,
                                      int sinks, int nk) {
    // first, last: places of the first and last row; keys past `last` are
    // seen by none
    hi = last + 1 < nk ? last + 1 : nk;
    lo = first >= window ? first - window + 1 : 0;
    sink_end = sinks < lo ? sinks : 0;
    if (sinks >= lo)
      lo = 0;
    if (hi < lo)
      hi = lo;
    sink_tiles = (sink_end + KT - 1) / KT;
    count = sink_tiles + (hi - lo + KT - 1) / KT;
  }
  __device__ __forceinline__ int from(int t) const {
    return t < sink_tiles ? t * KT : lo + (t - sink_tiles) * KT;
  }
  __device__ __forceinline__ int end(int t) const {
    return t < sink_tiles ? sink_end : hi;
  }
  __device__ __forceinline__ bool sink(int t) const { return t < sink_tiles; }
  // Whether rows at places lo .. hi each see every key of tile t,
  __device__ __forceinline__ bool all(int t, int place_lo, int place_hi,
                                      int window, int sinks) const {
    const int j = from(t), last = j + KT - 1;
    return sink(t) ? last < sink_end
                   : last <= place_lo &&
                         (place_hi - j < window || last < sinks);
  }
  // and whether one of them sees one.
  __device__ __forceinline__ bool any(int t, int place_lo, int place_hi,
                                      int window, int sinks) const {
    const int j = from(t), last = j + KT - 1;
    return sink(t) ||
           (j <= place_hi && (place_lo - last < window || j < sinks));
  }
};

// The key row in accumulator r of this lane, from the row block's start.
__device__ __forceinline__ int acc_row(int r) {
  return 8 * (r >> 2) + 4 * (lane_id() >> 5) + (r & 3);
}

// acc += A B where B's column is this lane's query and a key's row of B is
// zero for queries that do not see it.  Zero times an infinity or NaN of such
// a key would spoil the query's sum, so here every key is multiplied alone and
// added where it is seen (bit i of `seen`: the key of element i of this half of
// the wave; the halves' keys in turn).
template <typename T>
__device__ __forceinline__ v16f mma32_seen(Frag<T> a, Frag<T> b, v16f acc,
                                           uint32_t seen) {
  const int h = lane_id() >> 5;
  // the other half's verdicts on its own four keys each
  const auto sw =
      __builtin_amdgcn_permlane32_swap(seen, seen, false, false);
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const uint32_t bits = half ? sw[1] : sw[0];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const v16f one = mma32(one_of_frag<T>(a, i, h == half),
                             one_of_frag<T>(b, i, h == half), v16f{});
      const bool add = (bits >> i) & 1;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[r] += add ? one[r] : 0.0f;
    }
  }
  return acc;
}

// ---- forward -------------------------------------------------------------------

// The row kernels: STREAMS shares of the keys, each with tiles of its own that
// 4 / STREAMS waves of 32 rows go through.
template <typename T, int D, int STREAMS> struct Forward {
  static constexpr int kTile = sizeof(T) == 2 && STREAMS == 1 ? 64 : 32; // keys
  static constexpr int kBlocksOfRows = 4 / STREAMS;
  using Tile = RowTile<T, D, kTile, kThreads / STREAMS>;
  using Rows = ::Rows<shared_shift(STREAMS)>;
  static constexpr int kSteps = D / 16;   // products along d
  static constexpr int kBlocks = D / 32;  // output rows of 32
  static constexpr int kKeyBlocks = kTile / 32;
  static constexpr int kBytes = STREAMS * 4 * Tile::kBytes;
  // waves a SIMD: fp32 rows of 128 take more than half of the registers
  static constexpr int kWaves = sizeof(T) * D > 256 ? 1 : 2;
  static_assert(kBytes <= 128 * 1024, "");
};

// Adds up what the shares of the keys left in acc, in the first share's waves,
// share by share, under their common maximum; true in those waves.  acc and sum
// are 2^raise times smaller than the row's; they become `room` powers of two
// smaller still, so that adding keeps within fp32's range.  Every thread must
// call it, when the tiles' memory is free.
template <typename T, int D, int STREAMS, int BLOCKS>
__device__ __forceinline__ bool add_shares(v16f (&acc)[BLOCKS], float &top,
                                           float &sum, float &raise, float room,
                                           char *lds) {
  if constexpr (STREAMS == 1) {
    return true;
  } else {
    constexpr int kRowWords = BLOCKS * 16;
    constexpr int kWords = (kRowWords + 3) * kWave;
    constexpr int kRowBlocks = 4 / STREAMS;
    static_assert((4 - kRowBlocks) * kWords * 4 <=
                  Forward<T, D, STREAMS>::kBytes, "");
    const int wave = wave_in_group();
    float *words = reinterpret_cast<float *>(lds) + lane_id();
    __syncthreads();
    if (wave >= kRowBlocks) {
      float *x = words + (wave - kRowBlocks) * kWords;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[(b * 16 + r) * kWave] = acc[b][r];
      x[kRowWords * kWave] = top;
      x[(kRowWords + 1) * kWave] = sum;
      x[(kRowWords + 2) * kWave] = raise;
    }
    __syncthreads();
    if (wave >= kRowBlocks)
      return false;
#pragma unroll 1
    for (int i = 0; i < STREAMS - 1; ++i) {
      const float *x = words + (wave + i * kRowBlocks) * kWords;
      const float other = x[kRowWords * kWave];
      const float other_raise = x[(kRowWords + 2) * kWave];
      const float to = fmaxf(top, other);
      const float less = fmaxf(raise, other_raise) + room;
      const float by = (top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to)) *
                       __builtin_amdgcn_exp2f(raise - less);
      const float add =
          (other == to ? 1.0f : __builtin_amdgcn_exp2f(other - to)) *
          __builtin_amdgcn_exp2f(other_raise - less);
      top = to;
      raise = less;
      sum = fmaf(x[(kRowWords + 1) * kWave], add, sum * by);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          acc[b][r] = fmaf(x[(b * 16 + r) * kWave], add, acc[b][r] * by);
    }
    return true;
  }
}

// o and log_sum of a tile of rows, in one pass over the keys that they see.
// Matrix cores and the softmax's vector instructions bound it, the two waves
// of a SIMD taking turns: 65,536 queries, window 4096, 16 bf16 heads of 128
// take 2100 to 2210 us from card to card, 970 to 1020 TFLOP/s (a large matrix
// product of the library: 1170), the matrix cores half busy at 2.0 GHz; 16,384
// queries, window 1024, 32 heads 269 us.  Short calls wait for their chain of
// trips: 200 queries 7.1 us.
// A tile's scores computed under the softmax of the one before it, the wave's
// own turns overlapped, needs 32 registers more than there are: 2623 us.
template <typename T, int D, int STREAMS>
__global__ __launch_bounds__(kThreads, (Forward<T, D, STREAMS>::kWaves)) void
window_forward(WindowArgs a) {
  using F = Forward<T, D, STREAMS>;
  using Tile = typename F::Tile;
  constexpr int KT = F::kTile;
  __shared__ __align__(1024) char lds[F::kBytes];
  __shared__ int verdict;

  const int wave = wave_in_group();
  const int share = STREAMS == 1 ? 0 : wave / F::kBlocksOfRows;
  const int block = wave - share * F::kBlocksOfRows;
  const typename F::Rows w(a, block);
  if (w.count <= 0)
    return;
  const Sequence &s = w.s;
  const int lane = lane_id(), h = lane >> 5;
  const int place_lo = w.row_lo + w.shift, place_hi = place_lo + 31;
  const int row = w.row_lo + (lane & 31), place = row + w.shift;
  const bool live = row < s.nq;
  const int head = w.head, hk = w.key_head;

  // the wave's queries, negated where alpha is negative, and zero for an alpha of
  // zero, which would make a masked score of -inf a NaN
  const bool none = a.alpha == 0.0f;
  Frag<T> q[F::kSteps];
  load_rows<T>(q, static_cast<const T *>(a.query) +
                      (int64_t)(s.q0 + (live ? row : w.row0)) * a.q.token +
                      head * a.q.head, live && !none, a.d, a.alpha < 0.0f);
  const float scale = none ? 1.0f : fabsf(a.alpha) * kLog2e;

  const KeyTiles<KT> keys(w.row0 + w.shift, w.row0 + w.count - 1 + w.shift,
                          a.window, a.sinks, s.nk);
  const T *kbase = static_cast<const T *>(a.key) + (int64_t)s.k0 * a.k.token +
                   hk * a.k.head;
  const T *vbase = static_cast<const T *>(a.value) + (int64_t)s.k0 * a.v.token +
                   hk * a.v.head;
  const uint32_t kbytes = (uint32_t)(a.k.token * sizeof(T));
  const uint32_t vbytes = (uint32_t)(a.v.token * sizeof(T));
  typename Tile::Lane at;
  const uint32_t base = lds_address(lds) + share * 4 * Tile::kBytes;
  at.offset(base);
  // the share's tile of a step
  const int steps = (keys.count + STREAMS - 1) / STREAMS;
  auto copy = [&](int step) __attribute__((always_inline)) {
    const int t = step * STREAMS + share;
    if (t >= keys.count)
      return;
    const int64_t j = keys.from(t);
    const int n = keys.end(t) - (int)j;
    const uint32_t to = base + (step & 1) * 2 * Tile::kBytes;
    Tile::copy(to, kbase + j * a.k.token, n, kbytes, a.d, block);
    Tile::copy(to + Tile::kBytes, vbase + j * a.v.token, n, vbytes, a.d, block);
  };

  v16f acc[F::kBlocks];
  float top, sum;
  float raise = 0.0f; // of this lane's query, in the careful pass

  // One tile's products with the wave's queries.  Whole tiles are computed
  // where one of the rows sees a key: blocks of 32 keys apart, so that hidden
  // ones could be left out at the edges of the window, made the compiler move
  // the accumulators between two sets of registers (window 1024: 315 us
  // instead of 277).
  auto products = [&](uint32_t kt, int t, auto careful)
                      __attribute__((always_inline)) {
    constexpr int N = F::kKeyBlocks;
    const uint32_t vt = kt + Tile::kBytes;
    const bool all = keys.all(t, place_lo, place_hi, a.window, a.sinks);
    v16f score[N];
#pragma unroll
    for (int kb = 0; kb < N; ++kb)
      score[kb] = v16f{};
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st)
#pragma unroll
      for (int kb = 0; kb < N; ++kb)
        score[kb] = mma32(Tile::along(kt, at, kb, st), q[st], score[kb]);
    schedule_reads<sizeof(T) == 2 ? N * F::kSteps : 0>(); // (fp32: two reads each)
    uint32_t seen[N];
    if (!all) {
      // places before this lane's query (a sink tile's: any), and sinks left,
      // at the lane's first key
      const bool sink = keys.sink(t);
      const int j0 = keys.from(t) + 4 * h;
      const int back = sink ? 1 << 30 : place - j0;
      const uint32_t window = sink ? 0 : a.window;
      const int left = (sink ? keys.end(t) : a.sinks) - j0;
#pragma unroll
      for (int kb = 0; kb < N; ++kb) {
        seen[kb] = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = 32 * kb + 8 * (r >> 2) + (r & 3);
          const bool see = ((uint32_t)(back - j) < window) |
                           ((back >= j) & (left > j));
          score[kb][r] = see ? score[kb][r] : -kInf;
          if constexpr (decltype(careful)::value)
            seen[kb] |= (uint32_t)see << r;
        }
      }
    }
    // the running maximum follows a new one only past a factor of 2^8:
    // exp2(s - top) stays within fp32 and keeps its relative error
    float big = score[0][0];
#pragma unroll
    for (int kb = 0; kb < N; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        big = fmaxf(big, score[kb][r]);
    big = both_halves_max(big) * scale;
    if (ballot(big > top + 8.0f) != 0) {
      const float to = fmaxf(top, big);
      const float by = to == -kInf ? 1.0f : __builtin_amdgcn_exp2f(top - to);
      top = to;
      sum *= by;
#pragma unroll
      for (int b = 0; b < F::kBlocks; ++b)
        acc[b] *= by;
    }
    const float less = top == -kInf ? 0.0f : top;
    // (a factor of its own, so that the exponential keeps its bits)
    const float lower = __builtin_amdgcn_exp2f(-raise);
    // The wave that has come to its second product goes first: of two waves
    // of a SIMD one then multiplies while the other does its exponentials
    // (65,536 queries, window 4096: 2222 us without, 2167 us with)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kb = 0; kb < N; ++kb) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(fmaf(score[kb][r], scale, -less));
        if constexpr (decltype(careful)::value)
          p[r] *= lower;
        sum += p[r];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // bf16: the probabilities round to the operands' type, as the matrix
        // core takes them; their sum does not
        const Frag<T> pf = make_frag<T>(p + 8 * half);
#pragma unroll
        for (int b = 0; b < F::kBlocks; ++b) {
          const Frag<T> vf = Tile::across(vt, at, 2 * kb + half, b);
          if (decltype(careful)::value && !all)
            acc[b] = mma32_seen<T>(vf, pf, acc[b], seen[kb] >> (8 * half));
          else
            acc[b] = mma32(vf, pf, acc[b]);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  auto pass = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < F::kBlocks; ++b)
      acc[b] = v16f{};
    top = -kInf; // the largest scaled score, in powers of two
    sum = 0.0f;  // of this half's keys
    if (steps > 0)
      copy(0);
    // (the tile's place in LDS is a constant of each copy of the step, and so
    // are the addresses behind the lane's)
    auto step = [&](int i, auto parity) __attribute__((always_inline)) {
      landed();
      if (i + 1 < steps)
        copy(i + 1);
      const int t = i * STREAMS + share;
      if (t < keys.count &&
          keys.any(t, place_lo, place_hi, a.window, a.sinks))
        products(decltype(parity)::value * 2 * Tile::kBytes, t,
                 careful);
    };
    for (int i = 0; i < steps; i += 2) {
      step(i, std::integral_constant<int, 0>{});
      if (i + 1 < steps)
        step(i + 1, std::integral_constant<int, 1>{});
    }
  };
  pass(std::false_type{});
  // A finite result has met no infinity or NaN.  Others are computed again
  // with the keys at the edges of the mask kept apart.  A row that is not finite
  // may also be a sum past fp32's range of values whose mean lies within: its
  // probabilities, up to 2^8 of a lagging maximum, then are at most 2^(8 - raise),
  // so that no sum of them passes the largest value.  (Only in such a row: what
  // is below 2^(raise - 126) of the largest probability, or such a value, is
  // lost.)
  const bool finite = all_finite(acc);
  if (any_wave(!finite, &verdict)) {
    if (both_halves_max(finite ? 0.0f : 1.0f) != 0.0f)
      raise = 8.0f + raise_of(keys.count * KT);
    pass(std::true_type{});
  }

  if (!add_shares<T, D, STREAMS>(acc, top, sum, raise, 2.0f, lds))
    return;
  sum = both_halves_sum(sum);
  const bool empty = place < 0 || s.nk == 0; // a row that sees no key
  const float by = empty ? 0.0f : 1.0f / sum;
  if (live) {
    T *out = static_cast<T *>(a.output) + (int64_t)(s.q0 + row) * a.o.token +
             head * a.o.head;
#pragma unroll
    for (int b = 0; b < F::kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int c = 32 * b + acc_row(r);
        if (c < a.d)
          st4(out + c, empty ? 0.0f : acc[b][r] * by,
              empty ? 0.0f : acc[b][r + 1] * by,
              empty ? 0.0f : acc[b][r + 2] * by,
              empty ? 0.0f : acc[b][r + 3] * by);
      }
    if (a.log_sum && h == 0)
      a.log_sum[(int64_t)head * a.query_tokens + s.q0 + row] =
          empty ? -kInf
                : (top + __builtin_amdgcn_logf(
                             sum * __builtin_amdgcn_exp2f(raise))) * kLn2;
  }
}

// ---- backward ------------------------------------------------------------------

struct BackwardArgs {
  WindowArgs w; // o: the output's strides; log_sum: the forward pass's
  const void *output_gradient;
  void *query_gradient, *key_gradient, *value_gradient;
  Operand go, gq, gk, gv;
  float *log2_sum, *delta; // [query_heads][query_tokens], of the first kernel
  // Sums of the far sinks' gradients in fp32, [..][key_heads][32][2][d]: those
  // of the window for each block of 32 keys, and those of the queries past it,
  // for each block the ones of its sequence's first 1 << chunk_shift queries,
  // and behind them each later chunk's, sink_blocks of each.
  float *sink_window, *sink_chunks;
  float *part_sums; // [parts][split tiles][128][2][d]
  // Tiles of keys of all key heads: `whole` of them a workgroup each, the
  // `split` ones behind them `parts` each.
  int key_tiles, whole, split, parts;
  int chunks, chunk_shift;
  int far_blocks, sink_blocks; // blocks of all sequences, and the most of one
  int far_unit; // 0: far blocks are numbered by sequence; else window + 1
  bool far_by_key;
};

// A sequence's far sinks, those that a query sees from past its window: its
// first ones, as its last query stands at place nk - 1.
__device__ __forceinline__ int far_sinks(const WindowArgs &a,
                                         const Sequence &s) {
  const int n = s.nk - a.window < a.sinks ? s.nk - a.window : a.sinks;
  return n > 0 ? n : 0;
}
// The number of the first of a sequence's blocks of 32 far sinks, without a
// count of those before it.  Its u is its own among the sequences that have
// far sinks: its number, or, as these hold more than `window` keys each, its
// first key over window + 1.  A sequence's blocks are those from u sink_blocks
// on, or, by its first key, those from k0 / 32 + u on: fewer than 1 + f / 32
// of f far sinks, and k0 + f is at most the next one's first key.
__device__ __forceinline__ int first_far_block(const BackwardArgs &b, int i,
                                               int k0) {
  const int u = b.far_unit ? k0 / b.far_unit : i;
  return b.far_by_key ? (k0 >> 5) + u : u * b.sink_blocks;
}
// The sequence that far block n belongs to, where it belongs to one.
__device__ __forceinline__ int sequence_of_far_block(const BackwardArgs &b,
                                                     int n) {
  if (!b.far_unit && !b.far_by_key)
    return n / b.sink_blocks;
  return last_at_most(b.w.sequences, n, [&](int i) {
    return first_far_block(
        b, i, clamped(b.w.key_offsets[i], 0, b.w.key_tokens));
  });
}

// dq of a tile of rows, and for the second kernel log_sum in powers of two
// and delta of its rows.  The forward pass's loop with one product more:
// ds^T = K Q^T and V dO^T element by element, dq^T += K^T ds^T.  16,384 tokens,
// window 1024, 16 bf16 heads of 128 over 4: 233 us, the matrix cores 38 % busy
// (its rows of go leave no registers to read ahead).
template <typename T, int D, int STREAMS>
__global__ __launch_bounds__(kThreads, (Forward<T, D, STREAMS>::kWaves)) void
window_query_gradient(BackwardArgs b) {
  const WindowArgs &a = b.w;
  using F = Forward<T, D, STREAMS>;
  using Tile = typename F::Tile;
  constexpr int KT = F::kTile;
  __shared__ __align__(1024) char lds[F::kBytes];
  __shared__ int verdict;

  const int wave = wave_in_group();
  const int share = STREAMS == 1 ? 0 : wave / F::kBlocksOfRows;
  const int block = wave - share * F::kBlocksOfRows;
  const typename F::Rows w(a, block);
  if (w.count <= 0)
    return;
  const Sequence &s = w.s;
  const int lane = lane_id(), h = lane >> 5;
  const int place_lo = w.row_lo + w.shift, place_hi = place_lo + 31;
  const int row = w.row_lo + (lane & 31), place = row + w.shift;
  const bool live = row < s.nq;
  const int head = w.head, hk = w.key_head;
  const int64_t token = s.q0 + (live ? row : w.row0);

  const bool none = a.alpha == 0.0f;
  const float scale = none ? 1.0f : fabsf(a.alpha) * kLog2e;
  Frag<T> q[F::kSteps], go[F::kSteps];
  load_rows<T>(q, static_cast<const T *>(a.query) + token * a.q.token +
                      head * a.q.head, live && !none, a.d, a.alpha < 0.0f);
  load_rows<T>(go, static_cast<const T *>(b.output_gradient) +
                       token * b.go.token + head * b.go.head, live, a.d, false);
  float delta = 0.0f, log2_sum = 0.0f;
  {
    Frag<T> o[F::kSteps];
    load_rows<T>(o, static_cast<const T *>(a.output) + token * a.o.token +
                        head * a.o.head, live, a.d, false);
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st)
      delta = dot_frag<T>(go[st], o[st], delta);
    delta = both_halves_sum(delta);
    if (live) {
      const int64_t at = (int64_t)head * a.query_tokens + token;
      log2_sum = a.log_sum[at] * kLog2e;
      if (h == 0 && share == 0) {
        b.log2_sum[at] = log2_sum;
        b.delta[at] = delta;
      }
    }
  }

  const KeyTiles<KT> keys(w.row0 + w.shift, w.row0 + w.count - 1 + w.shift,
                          a.window, a.sinks, s.nk);
  const T *kbase = static_cast<const T *>(a.key) + (int64_t)s.k0 * a.k.token +
                   hk * a.k.head;
  const T *vbase = static_cast<const T *>(a.value) + (int64_t)s.k0 * a.v.token +
                   hk * a.v.head;
  const uint32_t kbytes = (uint32_t)(a.k.token * sizeof(T));
  const uint32_t vbytes = (uint32_t)(a.v.token * sizeof(T));
  typename Tile::FewLane at;
  const uint32_t base = lds_address(lds) + share * 4 * Tile::kBytes;
  at.offset(base);
  // the share's tile of a step
  const int steps = (keys.count + STREAMS - 1) / STREAMS;
  auto copy = [&](int step) __attribute__((always_inline)) {
    const int t = step * STREAMS + share;
    if (t >= keys.count)
      return;
    const int64_t j = keys.from(t);
    const int n = keys.end(t) - (int)j;
    const uint32_t to = base + (step & 1) * 2 * Tile::kBytes;
    Tile::copy(to, kbase + j * a.k.token, n, kbytes, a.d, block);
    Tile::copy(to + Tile::kBytes, vbase + j * a.v.token, n, vbytes, a.d, block);
  };

  v16f acc[F::kBlocks];
  auto products = [&](uint32_t kt, int t, auto careful)
                      __attribute__((always_inline)) {
    const uint32_t vt = kt + Tile::kBytes;
    at.fresh();
    const bool all = keys.all(t, place_lo, place_hi, a.window, a.sinks);
    const bool sink = keys.sink(t);
    const int j0 = keys.from(t) + 4 * h;
    const int back = sink ? 1 << 30 : place - j0;
    const uint32_t window = sink ? 0 : a.window;
    const int left = (sink ? keys.end(t) : a.sinks) - j0;
#pragma unroll
    for (int kb = 0; kb < F::kKeyBlocks; ++kb) {
      v16f p = {}, ds = {};
#pragma unroll
      for (int st = 0; st < F::kSteps; ++st) {
        p = mma32(Tile::along(kt, at, kb, st), q[st], p);
        ds = mma32(Tile::along(vt, at, kb, st), go[st], ds);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        ds[r] = __builtin_amdgcn_exp2f(fmaf(p[r], scale, -log2_sum)) *
                (ds[r] - delta);
      uint32_t seen = 0;
      if (!all) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = 32 * kb + 8 * (r >> 2) + (r & 3);
          const bool see = ((uint32_t)(back - j) < window) |
                           ((back >= j) & (left > j));
          ds[r] = see ? ds[r] : 0.0f;
          if constexpr (decltype(careful)::value)
            seen |= (uint32_t)see << r;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = ds[8 * half + i];
        // bf16: rounded once more, as the matrix core takes it
        const Frag<T> f = make_frag<T>(x);
#pragma unroll
        for (int c = 0; c < F::kBlocks; ++c) {
          const Frag<T> kf = Tile::across(kt, at, 2 * kb + half, c);
          if (decltype(careful)::value && !all)
            acc[c] = mma32_seen<T>(kf, f, acc[c], seen >> (8 * half));
          else
            acc[c] = mma32(kf, f, acc[c]);
        }
      }
    }
  };
  auto pass = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < F::kBlocks; ++c)
      acc[c] = v16f{};
    if (steps > 0)
      copy(0);
    auto step = [&](int i, auto parity) __attribute__((always_inline)) {
      landed();
      if (i + 1 < steps)
        copy(i + 1);
      const int t = i * STREAMS + share;
      if (t < keys.count &&
          keys.any(t, place_lo, place_hi, a.window, a.sinks))
        products(decltype(parity)::value * 2 * Tile::kBytes, t,
                 careful);
    };
    for (int i = 0; i < steps; i += 2) {
      step(i, std::integral_constant<int, 0>{});
      if (i + 1 < steps)
        step(i + 1, std::integral_constant<int, 1>{});
    }
  };
  pass(std::false_type{});
  if (any_wave(!all_finite(acc), &verdict))
    pass(std::true_type{});
  // (the shares' gradients add up as they are)
  float top = 0.0f, sum = 0.0f, raise = 0.0f;
  if (!add_shares<T, D, STREAMS>(acc, top, sum, raise, 0.0f, lds))
    return;
  if (live) {
    T *out = static_cast<T *>(b.query_gradient) + token * b.gq.token +
             head * b.gq.head;
#pragma unroll
    for (int c = 0; c < F::kBlocks; ++c)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        if (32 * c + acc_row(r) < a.d)
          st4(out + 32 * c + acc_row(r), acc[c][r] * a.alpha,
              acc[c][r + 1] * a.alpha, acc[c][r + 2] * a.alpha,
              acc[c][r + 3] * a.alpha);
  }
}

// dk and dv.  A workgroup holds 128 keys of one key head, 32 a wave, and goes
// through the queries that see them, head by head and 32 at a time: S = Q K^T
// and dP = dO V^T with queries in rows and keys in columns, dv^T += dO^T p,
// dk^T += Q^T ds.  K stays in registers and V in LDS: both in registers, and
// the sums, are more than two waves a SIMD have.
//
// The queries past the window that see the sinks are as many as the sequence
// has, so they are split (SINK): a workgroup of those takes 32 far sinks and a
// chunk of queries, its waves blocks of 32 queries in turn, each with tiles of
// its own, and leaves its sums to window_sink_gradient.
//
// Where there are few keys, or few behind a last full round of workgroups, the
// tiles of their queries are split into `parts`, one workgroup for each, whose
// sums window_key_join adds up.
//
// 16,384 tokens, window 1024, 16 bf16 heads of 128 over 4: 308 us, the matrix
// cores 35 % busy with four products a tile of 32 queries and one barrier (with
// K and V both in registers, one wave a SIMD: 603), and the sinks 31 us, a chain
// of few tiles: one wave a SIMD, the compiler having spilled 256 registers that
// its tiles' loop moves about, 4 of a block's 32 keys being sinks.
template <typename T, int D, bool SINK> struct Backward {
  static constexpr int kTile = 32; // queries
  using Tile = RowTile<T, D, kTile, SINK ? kWave : kThreads>;
  using Values = RowTile<T, D, kRows, kThreads>;
  static constexpr int kBuffers = SINK ? 4 : 1;
  // (fp32 rows of 128 leave a wave's own tiles no second place)
  static constexpr int kParities = SINK && sizeof(T) * D > 256 ? 1 : 2;
  static constexpr int kValues = SINK ? 0 : Values::kBytes;
  static constexpr int kBytes =
      kBuffers * kParities * 2 * Tile::kBytes + kValues;
  static constexpr int kSteps = D / 16;
  static constexpr int kBlocks = D / 32;
  static constexpr int kWaves = SINK || sizeof(T) * D > 256 ? 1 : 2;
};

// True: a sum is not finite, and nothing is written; CAREFUL computes those,
// with the queries at the edges of the mask kept apart.
template <typename T, int D, bool SINK, bool CAREFUL>
__device__ __forceinline__ bool key_gradient_rows(const BackwardArgs &b,
                                                  char *lds, float *stats,
                                                  int *verdict) {
  const WindowArgs &a = b.w;
  using F = Backward<T, D, SINK>;
  using Tile = typename F::Tile;
  using Values = typename F::Values;
  constexpr int QT = F::kTile;

  const int lane = lane_id(), h = lane >> 5, wave = wave_in_group();
  const int group = a.query_heads / a.key_heads;
  int hk, i, key0, first, last; // keys from key0; queries first .. last
  int far; // the sequence's far sinks
  Sequence s;
  int64_t item;
  int part = 0, parts = 1;
  if constexpr (SINK) {
    hk = blockIdx.x % a.key_heads;
    item = blockIdx.x / a.key_heads; // the block of sums
    int chunk = 0, least = 0;        // of the sequence's queries
    if (item < b.far_blocks) {
      i = sequence_of_far_block(b, (int)item);
      s = sequence(a, i);
      key0 = ((int)item - first_far_block(b, i, s.k0)) * 32;
    } else {
      // Later chunks of sequence i have the numbers from q0 >> chunk_shift on:
      // no more than whole chunks in its queries.
      const int x = ((int)item - b.far_blocks) / b.sink_blocks;
      key0 = ((int)item - b.far_blocks) % b.sink_blocks * 32;
      i = last_at_most(a.sequences, x, [&](int j) {
        return clamped(a.query_offsets[j], 0, a.query_tokens) >> b.chunk_shift;
      });
      s = sequence(a, i);
      chunk = x - (s.q0 >> b.chunk_shift) + 1;
      least = 1;
    }
    far = far_sinks(a, s);
    if (key0 < 0 || key0 >= far || chunk < least ||
        chunk > (s.nq - 1) >> b.chunk_shift)
      return false; // (none)
    first = chunk << b.chunk_shift;
    last = s.nq - 1 - first < 1 << b.chunk_shift
               ? s.nq - 1 : first + (1 << b.chunk_shift) - 1;
    if (last + s.nk - s.nq < a.window)
      return false; // (no query past the window: the sum leaves it out)
    const int past = key0 + a.window - (s.nk - s.nq);
    first = past > first ? past : first;
  } else {
    if ((int)blockIdx.x < b.whole) {
      item = xcd_contiguous(blockIdx.x, b.whole);
    } else {
      item = xcd_contiguous(blockIdx.x - b.whole, gridDim.x - b.whole);
      parts = b.parts;
      part = (int)(item % parts);
      item = b.whole + item / parts;
    }
    const int tile = (int)(item % b.key_tiles);
    hk = (int)(item / b.key_tiles);
    i = sequence_of_tile(a.key_offsets, a.sequences, tile, kRowShift);
    s = sequence(a, i);
    far = far_sinks(a, s);
    key0 = (tile - (a.key_offsets[i] >> kRowShift) - i) << kRowShift;
    if (key0 < 0 || key0 >= s.nk)
      return false;
    const int shift = s.nk - s.nq;
    const int end = (s.nk < key0 + kRows ? s.nk : key0 + kRows) - 1;
    first = key0 - shift > 0 ? key0 - shift : 0;
    last = s.nk - 1 - end < a.window ? s.nq - 1 : end + a.window - 1 - shift;
  }
  const int tile_key = key0;
  if constexpr (!SINK)
    key0 += 32 * wave;
  const int shift = s.nk - s.nq;
  const int key = key0 + (lane & 31);
  const bool live = key < (SINK ? far : s.nk);

  const bool none = a.alpha == 0.0f;
  const float scale = none ? 1.0f : fabsf(a.alpha) * kLog2e;
  const uint32_t vbase =
      lds_address(lds) + F::kBuffers * F::kParities * 2 * Tile::kBytes;
  Frag<T> k[F::kSteps], v[SINK ? F::kSteps : 1];
  {
    const int64_t token = s.k0 + (live ? key : 0);
    load_rows<T>(k, static_cast<const T *>(a.key) + token * a.k.token +
                        hk * a.k.head, live && !none, a.d, a.alpha < 0.0f);
    const T *values = static_cast<const T *>(a.value) + hk * a.v.head;
    if constexpr (SINK)
      load_rows<T>(v, values + token * a.v.token, live, a.d, false);
    else
      Values::copy(vbase, values + (int64_t)(s.k0 + tile_key) * a.v.token,
                   s.nk - tile_key, (uint32_t)(a.v.token * sizeof(T)), a.d,
                   wave);
  }

  const T *qbase = static_cast<const T *>(a.query) + (int64_t)s.q0 * a.q.token;
  const T *obase = static_cast<const T *>(b.output_gradient) +
                   (int64_t)s.q0 * b.go.token;
  const uint32_t qbytes = (uint32_t)(a.q.token * sizeof(T));
  const uint32_t obytes = (uint32_t)(b.go.token * sizeof(T));
  const int tiles = last < first ? 0 : (last - first) / QT + 1;
  // tiles of all heads, and this part's
  const int begin = SINK ? 0 : (int)((int64_t)tiles * group * part / parts);
  const int count =
      (SINK ? tiles * group
            : (int)((int64_t)tiles * group * (part + 1) / parts)) - begin;
  typename Tile::FewLane at;
  const uint32_t base =
      lds_address(lds) + (SINK ? wave * F::kParities * 2 * Tile::kBytes : 0);
  const uint32_t sbase = lds_address(stats) + (SINK ? wave * 1024 : 0);
  // the head and first query of the tile that is copied next, and of the one
  // that is computed next
  int next_head = 0, next = 0, now = 0;
  auto ahead = [&](int n) __attribute__((always_inline)) { // n tiles on
    next += n * QT;
    while (next > last) {
      next -= tiles * QT;
      ++next_head;
    }
  };
  if (count > 0) {
    next_head = hk * group + begin / tiles;
    next = first + begin % tiles * QT;
  }
  auto copy = [&](int parity) __attribute__((always_inline)) {
    const int head = next_head;
    const int64_t r = next;
    const int n = last + 1 - (int)r;
    const uint32_t to = base + parity * 2 * Tile::kBytes;
    Tile::copy(to, qbase + r * a.q.token + head * a.q.head, n, qbytes, a.d,
               SINK ? 0 : wave);
    Tile::copy(to + Tile::kBytes, obase + r * b.go.token + head * b.go.head, n,
               obytes, a.d, SINK ? 0 : wave);
    // a row's two numbers, 64 of each
    const int64_t row = (int64_t)head * a.query_tokens + s.q0 + r;
    const int m = n < QT ? n : QT;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (SINK || wave == e)
        copy_words_to_lds(
            buffer_words((e == 0 ? b.log2_sum : b.delta) + row, 4 * m),
            4 * lane, sbase + (parity * 2 + e) * 256);
  };

  v16f dk[F::kBlocks], dv[F::kBlocks];
  auto products = [&](int lo, int parity)
                      __attribute__((always_inline)) {
    const uint32_t qt = base + parity * 2 * Tile::kBytes;
    const uint32_t ot = qt + Tile::kBytes;
    const uint32_t st0 = sbase + parity * 512;
    if (!SINK &&
        (lo + 31 + shift < key0 || lo + shift - (key0 + 31) >= a.window))
      return; // hidden
    const bool all =
        lo + 31 <= last &&
        (SINK ? lo + shift - (key0 + 31) >= a.window && key0 + 32 <= far
              : lo + shift >= key0 + 31 && lo + 31 + shift - key0 < a.window);
    at.fresh();
    v16f p = {}, ds = {};
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st) {
      p = mma32(Tile::along(qt, at, 0, st), k[st], p);
      // (a tile of 128 rows has the lane's addresses of one of 32)
      if constexpr (SINK)
        ds = mma32(Tile::along(ot, at, 0, st), v[st], ds);
      else
        ds = mma32(Tile::along(ot, at, 0, st),
                   Tile::along(vbase + wave * 32 * Tile::kPitch, at, 0, st),
                   ds);
    }
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      // (rows acc_row(r) .. + 3 of the block)
      const v4f l4 = lds_read<v4f>(16 * h, st0 + 8 * r);
      const v4f d4 = lds_read<v4f>(16 * h, st0 + 256 + 8 * r);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[r + e] = __builtin_amdgcn_exp2f(fmaf(p[r + e], scale, -l4[e]));
        ds[r + e] = p[r + e] * (ds[r + e] - d4[e]);
      }
    }
    uint32_t seen = 0;
    if (!all) {
      const int back = lo + shift + 4 * h - key; // of accumulator row 0
      const int rows = last - lo - 4 * h;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 8 * (r >> 2) + (r & 3);
        const bool see =
            ((SINK ? (back + j >= a.window) & live
                   : (uint32_t)(back + j) < (uint32_t)a.window)) &
            (j <= rows);
        p[r] = see ? p[r] : 0.0f;
        ds[r] = see ? ds[r] : 0.0f;
        if constexpr (CAREFUL)
          seen |= (uint32_t)see << r;
      }
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = p[8 * half + e];
        y[e] = ds[8 * half + e];
      }
      // bf16: both round once more, as the matrix core takes them
      const Frag<T> pf = make_frag<T>(x), df = make_frag<T>(y);
#pragma unroll
      for (int c = 0; c < F::kBlocks; ++c) {
        const Frag<T> of = Tile::across(ot, at, half, c);
        const Frag<T> qf = Tile::across(qt, at, half, c);
        if (CAREFUL && !all) {
          dv[c] = mma32_seen<T>(of, pf, dv[c], seen >> (8 * half));
          dk[c] = mma32_seen<T>(qf, df, dk[c], seen >> (8 * half));
        } else {
          dv[c] = mma32(of, pf, dv[c]);
          dk[c] = mma32(qf, df, dk[c]);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  {
#pragma unroll
    for (int c = 0; c < F::kBlocks; ++c)
      dk[c] = dv[c] = v16f{};
    if constexpr (SINK) {
      if (wave < count)
        ahead(wave);
      if (wave < count && F::kParities == 2)
        copy(0);
      for (int t = wave, parity = 0; t < count; t += 4) {
        now = next;
        if (F::kParities == 1) {
          landed_wave(); // (its reads of the tile before)
          copy(0);
        }
        landed_wave();
        if (t + 4 < count) {
          ahead(4);
          if (F::kParities == 2)
            copy(parity ^ 1);
        }
        products(now, parity);
        parity ^= F::kParities - 1;
      }
    } else {
      if (count > 0)
        copy(0);
      auto step = [&](int t, auto parity) __attribute__((always_inline)) {
        constexpr int P = decltype(parity)::value;
        landed();
        now = next;
        if (t + 1 < count) {
          ahead(1);
          copy(1 - P);
        }
        products(now, P);
      };
      for (int t = 0; t < count; t += 2) {
        step(t, std::integral_constant<int, 0>{});
        if (t + 1 < count)
          step(t + 1, std::integral_constant<int, 1>{});
      }
    }
  }
  if (!CAREFUL && any_wave(!(all_finite(dk) && all_finite(dv)), verdict))
    return true;

  if constexpr (SINK) {
    // the waves' sums, one after the other, in the tiles' memory
    static_assert(F::kBytes >= 2 * F::kBlocks * 16 * 64 * 4, "");
    float *sums = reinterpret_cast<float *>(lds);
    for (int turn = 0; turn < 4; ++turn) {
      __syncthreads();
      if (turn == wave) {
#pragma unroll
        for (int c = 0; c < F::kBlocks; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float *x = sums + ((c * 16 + r) * 2) * 64 + lane;
            if (turn > 0) {
              dk[c][r] += x[0];
              dv[c][r] += x[64];
            }
            x[0] = dk[c][r];
            x[64] = dv[c][r];
          }
      }
    }
    if (wave != 3)
      return false;
  }
  if (!live)
    return false;
  // A part's sums wait for the other parts', and a far sink's for those of the
  // queries past the window.
  if (SINK || parts > 1 || key < far) {
    float *out;
    if (SINK)
      out = b.sink_chunks +
            ((item * a.key_heads + hk) * 32 + key - tile_key) * 2 * a.d;
    else if (parts > 1)
      out = b.part_sums + (((int64_t)part * b.split + item - b.whole) * kRows +
                           key - tile_key) * 2 * a.d;
    else
      out = b.sink_window +
            (((int64_t)(first_far_block(b, i, s.k0) + (key >> 5)) *
                  a.key_heads + hk) * 32 + (key & 31)) * 2 * a.d;
#pragma unroll
    for (int c = 0; c < F::kBlocks; ++c)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        if (32 * c + acc_row(r) < a.d) {
          float *x = out + 32 * c + acc_row(r);
          st4(x, dk[c][r], dk[c][r + 1], dk[c][r + 2], dk[c][r + 3]);
          st4(x + a.d, dv[c][r], dv[c][r + 1], dv[c][r + 2], dv[c][r + 3]);
        }
    return false;
  }
  const int64_t token = s.k0 + key;
  T *kout = static_cast<T *>(b.key_gradient) + token * b.gk.token +
            hk * b.gk.head;
  T *vout = static_cast<T *>(b.value_gradient) + token * b.gv.token +
            hk * b.gv.head;
#pragma unroll
  for (int c = 0; c < F::kBlocks; ++c)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      if (32 * c + acc_row(r) < a.d) {
        st4(kout + 32 * c + acc_row(r), dk[c][r] * a.alpha,
            dk[c][r + 1] * a.alpha, dk[c][r + 2] * a.alpha,
            dk[c][r + 3] * a.alpha);
        st4(vout + 32 * c + acc_row(r), dv[c][r], dv[c][r + 1], dv[c][r + 2],
            dv[c][r + 3]);
      }
  return false;
}

// CAREFUL is a function that is called and reads the kernel's arguments where
// they lie: inlined beside the plain one it takes registers of its loop, and a
// spilled register read back there waits for every copy under way (a training
// step of 16,384 tokens, window 1024: 707 us, inlined 752 us).
template <typename T, int D, bool SINK>
__device__ __noinline__ void key_gradient_again(const void *args, char *lds,
                                                float *stats, int *verdict) {
  key_gradient_rows<T, D, SINK, true>(*static_cast<const BackwardArgs *>(args),
                                      lds, stats, verdict);
}
template <typename T, int D, bool SINK>
__global__ __launch_bounds__(kThreads, (Backward<T, D, SINK>::kWaves)) void
window_key_gradient(BackwardArgs b) {
  using F = Backward<T, D, SINK>;
  // [buffer of a wave, or of all][parity][q, do], then the values
  __shared__ __align__(1024) char lds[F::kBytes];
  __shared__ __align__(16) float stats[F::kBuffers * 2 * 2 * 64];
  __shared__ int verdict;
  if (key_gradient_rows<T, D, SINK, false>(b, lds, stats, &verdict))
    key_gradient_again<T, D, SINK>(
        (const void *)__builtin_amdgcn_kernarg_segment_ptr(), lds, stats,
        &verdict);
}

// The far sinks' gradients: the window's sums, or its parts', and every chunk's,
// in the same order each time: eight runs of chunks, then the runs.  A workgroup
// of 128 x 8 threads for a far sink of one key head, 1 << shift of them a block; a
// launch and its trips to the sums: 64 chunks of 6 sequences, 4 sinks of 4 heads
// 4.2 us; 8 sequences of 64 sinks 10.5 us (with loops over a block's sinks and
// heads in one workgroup 14).
constexpr int kSinkRuns = 8;
template <typename T>
__global__ __launch_bounds__(128 * kSinkRuns) void
window_sink_gradient(BackwardArgs b, int shift) {
  const WindowArgs &a = b.w;
  __shared__ float sums[2][kSinkRuns][128];
  const int64_t id = block_id();
  const uint32_t item = (uint32_t)(id >> shift), heads = a.key_heads;
  const int hk = (int)(item % heads), block = (int)(item / heads);
  if (block >= b.far_blocks)
    return; // (a folded grid's last workgroups)
  const int i = sequence_of_far_block(b, block);
  const Sequence s = sequence(a, i);
  const int key0 = (block - first_far_block(b, i, s.k0)) * 32;
  const int row = (int)id & ((1 << shift) - 1), key = key0 + row;
  if (key0 < 0 || key >= far_sinks(a, s))
    return;
  const int run = threadIdx.x >> 7, c = threadIdx.x & 127;
  const int64_t size = (int64_t)a.key_heads * 32 * 2 * a.d; // floats of a block
  const int at = (hk * 32 + row) * 2 * a.d + c;             // in a block
  float dk = 0.0f, dv = 0.0f;
  if (c < a.d) {
    // chunks that reach past the window: those from the first whose last
    // query's place is at least a.window
    const int chunks = s.nq == 0 ? 0 : ((s.nq - 1) >> b.chunk_shift) + 1;
    const int past = a.window - (s.nk - s.nq); // query of that place
    int x = past <= 0 ? 0 : past >> b.chunk_shift;
    if (past > s.nq - 1)
      x = chunks; // (no query is past the window)
    // the sums of chunk 0 lie in this block, those of chunk x > 0 in
    // later + x sink_blocks
    const int64_t later = b.far_blocks + (key0 >> 5) +
                          ((int64_t)(s.q0 >> b.chunk_shift) - 1) *
                              b.sink_blocks;
    for (x += run; x < chunks; x += kSinkRuns) {
      const float *y =
          b.sink_chunks +
          (x == 0 ? block : later + (int64_t)x * b.sink_blocks) * size + at;
      dk += y[0];
      dv += y[a.d];
    }
  }
  sums[0][run][c] = dk;
  sums[1][run][c] = dv;
  __syncthreads();
  const int tile = (a.key_offsets[i] >> kRowShift) + i + (key >> kRowShift);
  if (run != 0 || c >= a.d || tile < 0 || tile >= b.key_tiles)
    return; // (tiles elsewhere: offsets outside the operands)
  dk = dv = 0.0f;
  const int64_t split = (int64_t)hk * b.key_tiles + tile - b.whole;
  const bool whole = split < 0;
  const float *x =
      whole ? b.sink_window + block * size + at
            : b.part_sums + (split * kRows + (key & (kRows - 1))) * 2 * a.d + c;
  const int64_t step = (int64_t)b.split * kRows * 2 * a.d;
  for (int p = 0; p < (whole ? 1 : b.parts); ++p) {
    dk += x[p * step];
    dv += x[p * step + a.d];
  }
#pragma unroll
  for (int r = 0; r < kSinkRuns; ++r) {
    dk += sums[0][r][c];
    dv += sums[1][r][c];
  }
  const int64_t token = s.k0 + key;
  stv(static_cast<T *>(b.key_gradient) + token * b.gk.token + hk * b.gk.head + c,
      dk * a.alpha);
  stv(static_cast<T *>(b.value_gradient) + token * b.gv.token +
          hk * b.gv.head + c, dv);
}

// The sums of the parts of the keys that are no far sinks, in order: four elements
// of a key and head a thread.  A launch and a trip, then memory: 3,001 tokens
// of 2 heads of 80 in 5 parts 5.5 us.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_key_join(BackwardArgs b) {
  const WindowArgs &a = b.w;
  const int per_row = a.d / 4;
  const int64_t x = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = x / per_row; // of the split tiles
  const int c = (int)(x % per_row) * 4;
  // (a tile has 128 rows of 2 and more threads: whole waves)
  const int64_t item =
      b.whole + __builtin_amdgcn_readfirstlane((int)(row >> kRowShift));
  const int tile = (int)(item % b.key_tiles), hk = (int)(item / b.key_tiles);
  const int i = sequence_of_tile(a.key_offsets, a.sequences, tile, kRowShift);
  const Sequence s = sequence(a, i);
  const int key0 = (tile - (a.key_offsets[i] >> kRowShift) - i) << kRowShift;
  const int key = key0 + (int)(row & (kRows - 1));
  if (key0 < 0 || key >= s.nk || key < far_sinks(a, s))
    return; // (none, or a far sink's)
  const int64_t token = s.k0 + key;
  const float *p = b.part_sums + row * 2 * a.d + c;
  const int64_t step = (int64_t)b.split * kRows * 2 * a.d;
  v4f dk = {}, dv = {};
#pragma unroll 4
  for (int i = 0; i < b.parts; ++i) {
    dk += ld4(p + i * step);
    dv += ld4(p + i * step + a.d);
  }
  st4(static_cast<T *>(b.key_gradient) + token * b.gk.token +
          hk * b.gk.head + c, dk[0] * a.alpha, dk[1] * a.alpha,
      dk[2] * a.alpha, dk[3] * a.alpha);
  st4(static_cast<T *>(b.value_gradient) + token * b.gv.token +
          hk * b.gv.head + c, dv[0], dv[1], dv[2], dv[3]);
}

// ---- host ------------------------------------------------------------------------

int check_window(int64_t sequences, int64_t query_tokens, int64_t key_tokens,
                 int64_t query_heads, int64_t key_heads, int64_t d,
                 int64_t window, int64_t sinks, float alpha) {
  if (sequences < 0 || query_tokens < 0 || key_tokens < 0 ||
      sequences > sw::kMostTokens || query_tokens > sw::kMostTokens ||
      key_tokens > sw::kMostTokens)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "expected 0 to 2^30 sequences and tokens, but got %lld, "
                    "%lld and %lld", (long long)sequences,
                    (long long)query_tokens, (long long)key_tokens);
  if (int rc = sw::check_heads(query_heads, key_heads, d))
    return rc;
  if (window < 1 || sinks < 0)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "expected a window of at least 1 and no negative sinks, "
                    "but got %lld and %lld", (long long)window,
                    (long long)sinks);
  // (scores are scaled by alpha log2 e)
  if (!std::isfinite(alpha * kLog2e))
    return sw::fail(SW_ERR_INVALID_ARGUMENT,
                    "alpha must be finite, and alpha log2 e too");
  return SW_OK;
}

// Checks what both directions take and fills `a`; `some` says whether there
// is anything to launch.
int fill_window(WindowArgs &a, size_t elem, const int32_t *query_offsets,
                const int32_t *key_offsets, const void *query, const void *key,
                const void *value, const void *output, const float *log_sum,
                int64_t sequences, int64_t query_tokens, int64_t key_tokens,
                int64_t query_heads, int64_t key_heads, int64_t d,
                const int64_t *strides, int64_t window, int64_t sinks,
                float alpha, bool writes) {
  if (int rc = check_window(sequences, query_tokens, key_tokens, query_heads,
                            key_heads, d, window, sinks, alpha))
    return rc;
  if (sequences > 0 && (!query_offsets || !key_offsets))
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "sequence offsets pointer is null");
  a.q = operand(strides, 0, query_heads, d);
  a.k = operand(strides, 1, key_heads, d);
  a.v = operand(strides, 2, key_heads, d);
  a.o = operand(strides, 3, query_heads, d);
  if (int rc = check_operand("query", query, a.q, d, elem, false, query_tokens,
                             query_heads))
    return rc;
  if (int rc = check_operand("key", key, a.k, d, elem, false, key_tokens,
                             key_heads))
    return rc;
  if (int rc = check_operand("value", value, a.v, d, elem, false, key_tokens,
                             key_heads))
    return rc;
  if (int rc = check_operand("output", output, a.o, d, elem, writes,
                             query_tokens, query_heads))
    return rc;
  if (int rc = sw::check_value_alignment(4, {query_offsets, key_offsets,
                                             log_sum}))
    return rc;
  a.query_offsets = query_offsets;
  a.key_offsets = key_offsets;
  a.query = query;
  a.key = key;
  a.value = value;
  a.output = const_cast<void *>(output);
  a.log_sum = const_cast<float *>(log_sum);
  a.sequences = (int)sequences;
  a.query_tokens = (int)query_tokens;
  a.key_tokens = (int)key_tokens;
  a.query_heads = (int)query_heads;
  a.key_heads = (int)key_heads;
  a.d = (int)d;
  // (no key lies past a window of all keys, so there are no sinks apart then)
  a.window = (int)std::min(window, std::max<int64_t>(key_tokens, 1));
  a.sinks = window >= key_tokens ? 0 : (int)std::min(sinks, key_tokens);
  a.alpha = alpha;
  return SW_OK;
}

// Shares of the keys for each workgroup of the row kernels.  The chip holds
// 512 workgroups (two waves a SIMD); about half of them and fewer are split.
// 4096 queries, window 1024, bf16 heads of 128, one share / two: 4 heads (132
// workgroups) 34.9 / 26.9 us, 8 heads (264) 39.5 / 36.0, 12 heads (396) 45.2 /
// 51.7, 32 heads (1056) 93.1 / 113.7; 2501 queries of 12 heads (288), window
// 2000: 63.9 / 72.8.  4, 8 and 12 heads of 64 in bf16 23.9 / 18.7, 24.6 / 21.3,
// 29.0 / 36.7, in fp32 93 / 52, 95 / 77, 151 / 147; fp32 heads of 128, of which
// the chip holds 256 workgroups, 167 / 101, 171 / 172, 332 / 257 (one number for
// all: 12 of these would gain).
int choose_streams(WindowArgs &a) {
  auto tiles = [&](int streams) {
    return ((int64_t)a.query_tokens >> shared_shift(streams)) + a.sequences;
  };
  const int streams = tiles(1) * a.query_heads < 272 ? 2 : 1;
  a.tiles = (int)tiles(streams);
  return streams;
}

template <typename T, int D>
int launch_forward(WindowArgs &a, int streams, hipStream_t st) {
  const int64_t grid = (int64_t)a.tiles * a.query_heads;
  if (int rc = sw::check_flat_grid(grid, kThreads, "window attention"))
    return rc;
  const dim3 g((unsigned)grid);
  if (streams == 1)
    window_forward<T, D, 1><<<g, kThreads, 0, st>>>(a);
  else
    window_forward<T, D, 2><<<g, kThreads, 0, st>>>(a);
  return sw::launch_check("window attention");
}

template <typename T>
int forward_entry(const int32_t *query_offsets, const int32_t *key_offsets,
                  const T *query, const T *key, const T *value, T *output,
                  float *log_sum, int64_t sequences, int64_t query_tokens,
                  int64_t key_tokens, int64_t query_heads, int64_t key_heads,
                  int64_t d, const int64_t *strides, int64_t window,
                  int64_t sinks, float alpha, void *stream) {
  sw::clear_error();
  WindowArgs a{};
  if (int rc = fill_window(a, sizeof(T), query_offsets, key_offsets, query, key,
                           value, output, log_sum, sequences, query_tokens,
                           key_tokens, query_heads, key_heads, d, strides,
                           window, sinks, alpha, true))
    return rc;
  if (sequences == 0 || query_tokens == 0)
    return SW_OK;
  const int streams = choose_streams(a);
  const hipStream_t st = sw::as_stream(stream);
  return d <= 64 ? launch_forward<T, 64>(a, streams, st)
                 : launch_forward<T, 128>(a, streams, st);
}

// The backward pass's scratch memory: [2][query_heads][query_tokens] of the
// queries' numbers, the sinks' sums, the parts' sums.
struct Scratch {
  int64_t stats, sink_window, sink_chunks, part_sums; // floats of each
  int64_t chunks, whole, split, far_blocks, sink_blocks, far_unit;
  int parts, chunk_shift, join_shift;
  bool far_by_key;
  int64_t bytes() const {
    return 4 * (2 * stats + sink_window + sink_chunks + part_sums);
  }
};
Scratch backward_scratch(int64_t sequences, int64_t query_tokens,
                         int64_t key_tokens, int64_t query_heads,
                         int64_t key_heads, int64_t d, int64_t window,
                         int64_t sinks, int64_t elem) {
  Scratch c{};
  // (whole 16 bytes, so that what follows stays aligned)
  c.stats = sw::ceil_div(query_heads * query_tokens, 4) * 4;
  // The chip holds 512 workgroups of 128 keys (256 of fp32 rows past 64).
  // Fewer are split until they are as many, as long as each part has eight
  // tiles of queries; a little more than half of them too, where a second part
  // of at least 32 tiles is worth its sums.  So are those behind the last full
  // round, unless they may be no more than the numbers between the sequences
  // that hold no keys.  4096 keys, window 1024, bf16 heads
  // of 128, one part / the rule's: 8 heads over 4 (132 workgroups) 164 / 100 us
  // (3 parts; 4: 128 us), 24 over 8 (264) 243 / 200 (2), 12 over 12 (396)
  // 115 (2 parts: 150).  The whole backward pass, window 1024 (fp32: 512), the
  // last round unsplit / split: 17,000 keys, bf16 heads of 128, 16 over 4 (532)
  // 702 / 573, 20,000 (628) 751 / 658, 16 over 16, 5120 keys (656) 231 / 219,
  // 4608 (592) 190 / 199; fp32 heads of 64, 16 over 8, 9000 keys (568)
  // 813 / 707; within the numbers without keys, 8192 (520) 579 / 617.  Forward
  // and backward in fp32, window 1024, one part / the rule's: 1000 tokens, 8
  // heads over 4 of 64 384 / 153 us, of 128 709 / 277; 4096 tokens, 8 over 4 of
  // 64 516 / 401, of 128 1017 / 1039, 24 over 8 of 64 1106 / 1068.
  const int64_t groups = ((key_tokens >> kRowShift) + sequences) * key_heads;
  const int64_t slots = elem == 4 && d > 64 ? 256 : 512;
  int64_t tail = groups % slots;
  if (groups > slots && tail <= sequences * key_heads)
    tail = 0;
  const int64_t tiles = query_heads / key_heads *
                        (std::min({window, key_tokens, query_tokens}) + kRows) /
                        32;
  int64_t parts = tail == 0 ? 1 : std::min(slots / tail, tiles / 8);
  if (parts == 1 && tail * 8 <= slots * 5 && tiles >= 64)
    parts = 2;
  c.parts = (int)std::max<int64_t>(1, std::min<int64_t>(parts, 16));
  c.split = c.parts > 1 ? tail : 0;
  c.whole = groups - c.split;
  c.part_sums = c.split * c.parts * kRows * 2 * d;
  // A sequence's far sinks: no more than its keys but `window`.
  const int64_t s =
      window >= key_tokens ? 0 : std::min(sinks, key_tokens - window);
  if (s == 0)
    return c;
  // Their blocks by sequence, which needs no search, unless that makes more
  // rows than there are keys: sequences that are shorter than the sinks are
  // many, or few hold more than `window` keys.
  c.sink_blocks = sw::ceil_div(s, 32);
  c.far_blocks = sequences * c.sink_blocks;
  if (c.far_blocks * 32 > key_tokens) {
    const int64_t units = key_tokens / (window + 1);
    c.far_unit = units < sequences ? window + 1 : 0;
    const int64_t by_unit = std::min(sequences, units) * c.sink_blocks;
    const int64_t by_key =
        (key_tokens - window) / 32 + std::min(sequences, units);
    c.far_by_key = by_key < by_unit;
    c.far_blocks = std::min(by_key, by_unit);
  }
  // 256 queries a chunk, more where there are more than 64 sinks: the sums of
  // all but the sequences' first chunks then have at most a row for four
  // queries, the size of bf16 keys; fewer, to 64, where that makes fewer
  // workgroups than the chip has units.
  c.chunk_shift = 8;
  while (((int64_t)64 << (c.chunk_shift - 8)) < s && c.chunk_shift < 30)
    ++c.chunk_shift;
  while (c.chunk_shift > 6 &&
         ((query_tokens >> c.chunk_shift) * c.sink_blocks + c.far_blocks) *
                 key_heads < 256)
    --c.chunk_shift;
  c.chunks = query_tokens >> c.chunk_shift;
  // places for a block's far sinks in the join's grid
  while (c.join_shift < 5 && ((int64_t)1 << c.join_shift) < s)
    ++c.join_shift;
  const int64_t one = key_heads * 32 * 2 * d;
  c.sink_window = c.far_blocks * one;
  c.sink_chunks = (c.far_blocks + c.chunks * c.sink_blocks) * one;
  return c;
}

template <typename T, int D>
int launch_backward(BackwardArgs &b, int join_shift, hipStream_t st) {
  WindowArgs &a = b.w;
  const char *what = "window attention's gradient";
  const int streams = choose_streams(a);
  const int64_t rows = (int64_t)a.tiles * a.query_heads;
  const int64_t sinks =
      (b.far_blocks + (int64_t)b.chunks * b.sink_blocks) * a.key_heads;
  const int64_t keys = (int64_t)b.key_tiles * a.key_heads +
                       (int64_t)b.split * (b.parts - 1);
  const int64_t part_rows = (int64_t)b.split * kRows * (a.d / 4) / kThreads;
  const int64_t join = ((int64_t)b.far_blocks * a.key_heads) << join_shift;
  if (int rc = sw::check_flat_grid(std::max({rows, sinks, keys, part_rows}),
                                   kThreads, what))
    return rc;
  if (int rc = sw::check_grid(join, 128 * kSinkRuns, what))
    return rc;
  if (a.query_tokens > 0) {
    const dim3 g((unsigned)rows);
    if (streams == 1)
      window_query_gradient<T, D, 1><<<g, kThreads, 0, st>>>(b);
    else
      window_query_gradient<T, D, 2><<<g, kThreads, 0, st>>>(b);
    if (int rc = sw::launch_check(what))
      return rc;
  }
  if (a.key_tokens == 0)
    return SW_OK;
  if (sinks > 0) {
    window_key_gradient<T, D, true>
        <<<dim3((unsigned)sinks), kThreads, 0, st>>>(b);
    if (int rc = sw::launch_check(what))
      return rc;
  }
  window_key_gradient<T, D, false>
      <<<dim3((unsigned)keys), kThreads, 0, st>>>(b);
  if (int rc = sw::launch_check(what))
    return rc;
  if (part_rows > 0) {
    window_key_join<T><<<dim3((unsigned)part_rows), kThreads, 0, st>>>(b);
    if (int rc = sw::launch_check(what))
      return rc;
  }
  if (b.far_blocks > 0) {
    window_sink_gradient<T><<<sw::grid_dim(join, 128 * kSinkRuns),
                              128 * kSinkRuns, 0, st>>>(b, join_shift);
    return sw::launch_check(what);
  }
  return SW_OK;
}

template <typename T>
int backward_entry(const int32_t *query_offsets, const int32_t *key_offsets,
                   const T *query, const T *key, const T *value,
                   const T *output, const float *log_sum,
                   const T *output_gradient, T *query_gradient,
                   T *key_gradient, T *value_gradient, int64_t sequences,
                   int64_t query_tokens, int64_t key_tokens,
                   int64_t query_heads, int64_t key_heads, int64_t d,
                   const int64_t *strides, int64_t window, int64_t sinks,
                   float alpha, void *workspace, int64_t workspace_bytes,
                   void *stream) {
  sw::clear_error();
  BackwardArgs b{};
  WindowArgs &a = b.w;
  if (int rc = fill_window(a, sizeof(T), query_offsets, key_offsets, query, key,
                           value, output, log_sum, sequences, query_tokens,
                           key_tokens, query_heads, key_heads, d, strides,
                           window, sinks, alpha, false))
    return rc;
  b.go = operand(strides, 4, query_heads, d);
  b.gq = operand(strides, 5, query_heads, d);
  b.gk = operand(strides, 6, key_heads, d);
  b.gv = operand(strides, 7, key_heads, d);
  if (int rc = check_operand("output gradient", output_gradient, b.go, d,
                             sizeof(T), false, query_tokens, query_heads))
    return rc;
  if (int rc = check_operand("query gradient", query_gradient, b.gq, d,
                             sizeof(T), true, query_tokens, query_heads))
    return rc;
  if (int rc = check_operand("key gradient", key_gradient, b.gk, d, sizeof(T),
                             true, key_tokens, key_heads))
    return rc;
  if (int rc = check_operand("value gradient", value_gradient, b.gv, d,
                             sizeof(T), true, key_tokens, key_heads))
    return rc;
  if (sequences == 0 || (query_tokens == 0 && key_tokens == 0))
    return SW_OK;
  if (!log_sum && query_tokens > 0)
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "log_sum pointer is null");
  const Scratch c = backward_scratch(sequences, query_tokens, key_tokens,
                                     query_heads, key_heads, d, window, sinks,
                                     sizeof(T));
  if (c.bytes() > 0 && (!workspace || !sw::aligned16(workspace) ||
                        workspace_bytes < c.bytes()))
    return sw::fail(SW_ERR_INVALID_ARGUMENT,
                    "the backward pass needs a 16-byte aligned workspace of "
                    "%lld bytes", (long long)c.bytes());
  b.output_gradient = output_gradient;
  b.query_gradient = query_gradient;
  b.key_gradient = key_gradient;
  b.value_gradient = value_gradient;
  b.log2_sum = static_cast<float *>(workspace);
  b.delta = b.log2_sum + c.stats;
  b.sink_window = b.delta + c.stats;
  b.sink_chunks = b.sink_window + c.sink_window;
  b.chunks = (int)c.chunks;
  b.chunk_shift = c.chunk_shift;
  b.far_blocks = (int)c.far_blocks;
  b.sink_blocks = (int)c.sink_blocks;
  b.far_unit = (int)c.far_unit;
  b.far_by_key = c.far_by_key;
  b.part_sums = b.sink_chunks + c.sink_chunks;
  b.parts = c.parts;
  b.whole = (int)c.whole;
  b.split = (int)c.split;
  b.key_tiles = (int)((key_tokens >> kRowShift) + sequences);
  const hipStream_t st = sw::as_stream(stream);
  return d <= 64 ? launch_backward<T, 64>(b, c.join_shift, st)
                 : launch_backward<T, 128>(b, c.join_shift, st);
}

} // namespace

extern "C" int sw_window_attention_f32(
    const int32_t *query_offsets, const int32_t *key_offsets,
    const float *query, const float *key, const float *value, float *output,
    float *log_sum, int64_t sequences, int64_t query_tokens,
    int64_t key_tokens, int64_t query_heads, int64_t key_heads, int64_t d,
    const int64_t *strides, int64_t window, int64_t sinks, float alpha,
    void *stream) {
  return forward_entry<float>(query_offsets, key_offsets, query, key, value,
                              output, log_sum, sequences, query_tokens,
                              key_tokens, query_heads, key_heads, d, strides,
                              window, sinks, alpha, stream);
}

extern "C" int sw_window_attention_bf16(
    const int32_t *query_offsets, const int32_t *key_offsets,
    const uint16_t *query, const uint16_t *key, const uint16_t *value,
    uint16_t *output, float *log_sum, int64_t sequences, int64_t query_tokens,
    int64_t key_tokens, int64_t query_heads, int64_t key_heads, int64_t d,
    const int64_t *strides, int64_t window, int64_t sinks, float alpha,
    void *stream) {
  return forward_entry<uint16_t>(query_offsets, key_offsets, query, key, value,
                                 output, log_sum, sequences, query_tokens,
                                 key_tokens, query_heads, key_heads, d,
                                 strides, window, sinks, alpha, stream);
}

extern "C" int64_t sw_window_attention_backward_workspace_bytes(
    int64_t sequences, int64_t query_tokens, int64_t key_tokens,
    int64_t query_heads, int64_t key_heads, int64_t d, int64_t window,
    int64_t sinks, int value_bytes) {
  if ((value_bytes != 4 && value_bytes != 2) ||
      check_window(sequences, query_tokens, key_tokens, query_heads, key_heads,
                   d, window, sinks, 0.0f) != SW_OK)
    return 0;
  return backward_scratch(sequences, query_tokens, key_tokens, query_heads,
                          key_heads, d, window, sinks, value_bytes).bytes();
}

extern "C" int sw_window_attention_backward_f32(
    const int32_t *query_offsets, const int32_t *key_offsets,
    const float *query, const float *key, const float *value,
    const float *output, const float *log_sum, const float *output_gradient,
    float *query_gradient, float *key_gradient, float *value_gradient,
    int64_t sequences, int64_t query_tokens, int64_t key_tokens,
    int64_t query_heads, int64_t key_heads, int64_t d, const int64_t *strides,
    int64_t window, int64_t sinks, float alpha, void *workspace,
    int64_t workspace_bytes, void *stream) {
  return backward_entry<float>(
      query_offsets, key_offsets, query, key, value, output, log_sum,
      output_gradient, query_gradient, key_gradient, value_gradient, sequences,
      query_tokens, key_tokens, query_heads, key_heads, d, strides, window,
      sinks, alpha, workspace, workspace_bytes, stream);
}

extern "C" int sw_window_attention_backward_bf16(
    const int32_t *query_offsets, const int32_t *key_offsets,
    const uint16_t *query, const uint16_t *key, const uint16_t *value,
    const uint16_t *output, const float *log_sum,
    const uint16_t *output_gradient, uint16_t *query_gradient,
    uint16_t *key_gradient, uint16_t *value_gradient, int64_t sequences,
    int64_t query_tokens, int64_t key_tokens, int64_t query_heads,
    int64_t key_heads, int64_t d, const int64_t *strides, int64_t window,
    int64_t sinks, float alpha, void *workspace, int64_t workspace_bytes,
    void *stream) {
  return backward_entry<uint16_t>(
      query_offsets, key_offsets, query, key, value, output, log_sum,
      output_gradient, query_gradient, key_gradient, value_gradient, sequences,
      query_tokens, key_tokens, query_heads, key_heads, d, strides, window,
      sinks, alpha, workspace, workspace_bytes, stream);
}
