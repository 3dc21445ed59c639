// Attention over a sliding window with sinks, forward and backward, for packed
// sequences on gfx950.
//
// Query i of a sequence of nq queries and nk keys stands at p = i + nk - nq
// and sees key j where j <= p and (p - j < window or j < sinks):
//   s = alpha q.k,  m = max s,  l = sum exp(s - m),
//   o = sum exp(s - m) v / l,  log_sum = m + log l.
// Query heads g G .. g G + G - 1 share key head g, G = query_heads / key_heads.
#include "sw_heads.h"
#include "sw_internal.h"

#include <algorithm>
#include <cmath>

using namespace swd;

namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kInf = __builtin_inff();

constexpr int kThreads = 256; // four waves of 32 rows
constexpr int kRowShift = 7;
constexpr int kRows = 1 << kRowShift;

struct Operand {
  int64_t token, head; // strides in elements
};

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
// added where it is seen (bit i of `seen`: the key of element i of this half;
// `mine` / `other` halves in turn).
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

template <typename T, int D> struct Forward {
  static constexpr int kTile = sizeof(T) == 2 ? 64 : 32; // keys
  using Tile = RowTile<T, D, kTile, kThreads>;
  static constexpr int kSteps = D / 16;   // products along d
  static constexpr int kBlocks = D / 32;  // output rows of 32
  static constexpr int kKeyBlocks = kTile / 32;
  // waves a SIMD: fp32 rows of 128 take more than half of the registers
  static constexpr int kWaves = sizeof(T) * D > 256 ? 1 : 2;
};

template <typename T, int D>
__global__ __launch_bounds__(kThreads, (Forward<T, D>::kWaves)) void
window_forward(WindowArgs a) {
  using F = Forward<T, D>;
  using Tile = typename F::Tile;
  constexpr int KT = F::kTile;
  __shared__ __align__(1024) char lds[2][2][Tile::kBytes];
  __shared__ int spoiled;

  const int group = a.query_heads / a.key_heads;
  int64_t item = xcd_contiguous(blockIdx.x, gridDim.x);
  const int g = (int)(item % group);
  item /= group;
  const int tile = (int)(item % a.tiles);
  const int hk = (int)(item / a.tiles);
  const int head = hk * group + g;

  const int seq = sequence_of_tile(a.query_offsets, a.sequences, tile, kRowShift);
  const Sequence s = sequence(a, seq);
  const int row0 =
      (tile - (a.query_offsets[seq] >> kRowShift) - seq) << kRowShift;
  if (row0 < 0 || row0 >= s.nq)
    return;
  const int rows = s.nq - row0 < kRows ? s.nq - row0 : kRows;
  const int shift = s.nk - s.nq; // a query's place less its index

  const int lane = lane_id(), h = lane >> 5, wave = wave_in_group();
  const int row = row0 + 32 * wave + (lane & 31);
  const bool live = row < s.nq;
  const int place = row + shift;
  const int place_lo = row0 + 32 * wave + shift, place_hi = place_lo + 31;

  // the wave's queries, negated where alpha is negative, and zero for an alpha
  // too small to scale a masked score of -inf
  Frag<T> q[F::kSteps];
  const bool tiny = fabsf(a.alpha) < 0x1p-126f;
  {
    const T *p = static_cast<const T *>(a.query) +
                 (int64_t)(s.q0 + (live ? row : row0)) * a.q.token +
                 head * a.q.head;
#pragma unroll
    for (int st = 0; st < F::kSteps; ++st) {
      const int c = 16 * st + 8 * h;
      q[st] = live && c < a.d && !tiny ? ld_frag(p + c) : zero_frag<T>();
      if (a.alpha < 0.0f)
        q[st] = negate_frag<T>(q[st]);
    }
  }
  const float scale = tiny ? 1.0f : fabsf(a.alpha) * kLog2e;

  const KeyTiles<KT> keys(row0 + shift, row0 + rows - 1 + shift, a.window,
                          a.sinks, s.nk);
  const T *kbase = static_cast<const T *>(a.key) + (int64_t)s.k0 * a.k.token +
                   hk * a.k.head;
  const T *vbase = static_cast<const T *>(a.value) + (int64_t)s.k0 * a.v.token +
                   hk * a.v.head;
  const uint32_t kbytes = (uint32_t)(a.k.token * sizeof(T));
  const uint32_t vbytes = (uint32_t)(a.v.token * sizeof(T));
  const typename Tile::Lane at;
  const uint32_t base = lds_address(lds);
  auto copy = [&](int t) __attribute__((always_inline)) {
    const int64_t j = keys.from(t);
    const int n = keys.end(t) - (int)j;
    const uint32_t to = base + (t & 1) * 2 * Tile::kBytes;
    Tile::copy(to, kbase + j * a.k.token, n, kbytes, a.d);
    Tile::copy(to + Tile::kBytes, vbase + j * a.v.token, n, vbytes, a.d);
  };

  v16f acc[F::kBlocks];
  float top, sum;

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
    for (int kb = 0; kb < N; ++kb) {
      score[kb] = v16f{};
#pragma unroll
      for (int st = 0; st < F::kSteps; ++st)
        score[kb] = mma32(Tile::along(kt, at, kb, st), q[st], score[kb]);
    }
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
    if (keys.count > 0)
      copy(0);
    // (the tile's place in LDS is a constant of each copy of the step, and so
    // are the addresses behind the lane's)
    auto step = [&](int t, auto parity) __attribute__((always_inline)) {
      landed();
      if (t + 1 < keys.count)
        copy(t + 1);
      if (keys.any(t, place_lo, place_hi, a.window, a.sinks))
        products(base + decltype(parity)::value * 2 * Tile::kBytes, t,
                 careful);
    };
    for (int t = 0; t < keys.count; t += 2) {
      step(t, std::integral_constant<int, 0>{});
      if (t + 1 < keys.count)
        step(t + 1, std::integral_constant<int, 1>{});
    }
  };
  pass(std::false_type{});
  // A finite result has met no infinity or NaN.  Others are computed again
  // with the keys at the edges of the mask kept apart.
  {
    float x = 0.0f;
#pragma unroll
    for (int b = 0; b < F::kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        x = fmaf(acc[b][r], 0.0f, x);
    if (threadIdx.x == 0)
      spoiled = 0;
    __syncthreads();
    if (ballot(x != 0.0f) != 0 && lane == 0)
      spoiled = 1;
    __syncthreads();
    if (spoiled)
      pass(std::true_type{});
  }

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
          empty ? -kInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

// ---- host ------------------------------------------------------------------------

// Strides of one operand: rows of d elements, 16-byte aligned, close enough
// that a tile of rows spans 2^30 bytes (descriptor offsets are 32 bits).
int check_operand(const char *name, const void *p, const Operand &s, int64_t d,
                  int64_t elem, bool some, bool output, int64_t tokens,
                  int64_t heads) {
  if (!some)
    return SW_OK;
  if (!p)
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "%s pointer is null", name);
  if (!sw::aligned16(p) || s.token * elem % 16 != 0 || s.head * elem % 16 != 0)
    return sw::fail(SW_ERR_INVALID_ARGUMENT,
                    "%s must be 16-byte aligned, its strides included", name);
  if (s.token < d || s.head < 0 || s.token * elem > (int64_t)1 << 23)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "%s strides must be at least d = %lld (tokens; at most "
                    "2^23 bytes) and 0 (heads), but got %lld and %lld",
                    name, (long long)d, (long long)s.token, (long long)s.head);
  if (output && heads > 1) {
    // heads within a token's row, or a head's tokens within its plane
    const bool in_row = s.head >= d && s.token >= (heads - 1) * s.head + d;
    const bool in_plane = s.head >= (tokens - 1) * s.token + d;
    if (!in_row && !in_plane)
      return sw::fail(SW_ERR_INVALID_SHAPE, "%s rows overlap", name);
  }
  return SW_OK;
}

constexpr int64_t kMostTokens = (int64_t)1 << 30;

Operand operand(const int64_t *strides, int i, int64_t heads, int64_t d) {
  if (strides)
    return {strides[2 * i], strides[2 * i + 1]};
  return {heads * d, d};
}

int check_window(int64_t sequences, int64_t query_tokens, int64_t key_tokens,
                 int64_t query_heads, int64_t key_heads, int64_t d,
                 int64_t window, int64_t sinks, float alpha) {
  if (sequences < 0 || query_tokens < 0 || key_tokens < 0 ||
      sequences > kMostTokens || query_tokens > kMostTokens ||
      key_tokens > kMostTokens)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "expected 0 to 2^30 sequences and tokens, but got %lld, "
                    "%lld and %lld", (long long)sequences,
                    (long long)query_tokens, (long long)key_tokens);
  if (query_heads < 1 || key_heads < 1 || query_heads > 65536 ||
      query_heads % key_heads != 0)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "query heads must be a multiple of key heads (at most "
                    "65536), but got %lld and %lld", (long long)query_heads,
                    (long long)key_heads);
  if (d < 8 || d > 128 || d % 8 != 0)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "head dimension must be a multiple of 8 up to 128, but "
                    "got %lld", (long long)d);
  if (window < 1 || sinks < 0)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "expected a window of at least 1 and no negative sinks, "
                    "but got %lld and %lld", (long long)window,
                    (long long)sinks);
  if (!std::isfinite(alpha))
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "alpha must be finite");
  return SW_OK;
}

template <typename T>
int forward_entry(const int32_t *query_offsets, const int32_t *key_offsets,
                  const T *query, const T *key, const T *value, T *output,
                  float *log_sum, int64_t sequences, int64_t query_tokens,
                  int64_t key_tokens, int64_t query_heads, int64_t key_heads,
                  int64_t d, const int64_t *strides, int64_t window,
                  int64_t sinks, float alpha, void *stream) {
  sw::clear_error();
  if (int rc = check_window(sequences, query_tokens, key_tokens, query_heads,
                            key_heads, d, window, sinks, alpha))
    return rc;
  if (sequences > 0 && (!query_offsets || !key_offsets))
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "sequence offsets pointer is null");
  WindowArgs a{};
  a.q = operand(strides, 0, query_heads, d);
  a.k = operand(strides, 1, key_heads, d);
  a.v = operand(strides, 2, key_heads, d);
  a.o = operand(strides, 3, query_heads, d);
  if (int rc = check_operand("query", query, a.q, d, sizeof(T), query_tokens > 0, false, query_tokens, query_heads))
    return rc;
  if (int rc = check_operand("key", key, a.k, d, sizeof(T), key_tokens > 0, false, key_tokens, key_heads))
    return rc;
  if (int rc = check_operand("value", value, a.v, d, sizeof(T), key_tokens > 0, false, key_tokens, key_heads))
    return rc;
  if (int rc = check_operand("output", output, a.o, d, sizeof(T), query_tokens > 0, true, query_tokens, query_heads))
    return rc;
  if (int rc = sw::check_value_alignment(4, {log_sum}))
    return rc;
  if (sequences == 0 || query_tokens == 0)
    return SW_OK;
  a.query_offsets = query_offsets;
  a.key_offsets = key_offsets;
  a.query = query;
  a.key = key;
  a.value = value;
  a.output = output;
  a.log_sum = log_sum;
  a.sequences = (int)sequences;
  a.query_tokens = (int)query_tokens;
  a.key_tokens = (int)key_tokens;
  a.query_heads = (int)query_heads;
  a.key_heads = (int)key_heads;
  a.d = (int)d;
  a.window = (int)std::min(window, std::max<int64_t>(key_tokens, 1));
  a.sinks = (int)std::min(sinks, key_tokens);
  a.alpha = alpha;
  const int64_t tiles = (query_tokens >> kRowShift) + sequences;
  a.tiles = (int)tiles;
  const int64_t grid = tiles * query_heads;
  if (int rc = sw::check_flat_grid(grid, kThreads, "window attention"))
    return rc;
  const hipStream_t st = sw::as_stream(stream);
  if (d <= 64)
    window_forward<T, 64><<<dim3((unsigned)grid), kThreads, 0, st>>>(a);
  else
    window_forward<T, 128><<<dim3((unsigned)grid), kThreads, 0, st>>>(a);
  return sw::launch_check("window attention");
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
