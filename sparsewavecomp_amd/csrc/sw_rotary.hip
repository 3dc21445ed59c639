// Rotary positions: pairs of each head's elements turned by an angle,
//   (x, y) -> (x cos t - y sin t, x sin t + y cos t),
//   t = positions[axis of the pair][token] frequency of the pair,
// the pairs being elements i and i + pairs of a head, or 2 i and 2 i + 1; the
// gradients are turned by -t.
//
// Each element is read and written once, three operations for it: memory bounds
// this (32,760 tokens of 40 heads of 128, bf16, three axes, 671 MB: 109 us, 6.1
// TB/s; 16,384 of 20, 168 MB: 26, 6.5; a large copy reaches 6.3; 64 tokens: 3.5).
// The angles belong to a token and are shared by its heads, so a
// workgroup computes those of its tokens first.  They are reduced to a quarter
// turn in 64 bits: a position of 2^17 times a frequency near 1 has lost 2^-8 of
// a radian in 32.
#include "sw_heads.h"
#include "sw_internal.h"

#include <algorithm>
#include <type_traits>

using namespace swd;
using sw::check_operand;

namespace {

constexpr int kThreads = 256;

struct Heads {
  const void *from;
  void *to;
  int64_t from_token, from_head, to_token, to_head; // strides in elements
};

struct RotaryArgs {
  const int32_t *positions, *axes; // axes may be null: all pairs take axis 0
  const float *frequencies;
  Heads query, key;
  int tokens, axis_count, query_heads, heads, d, pairs;
  int per; // tokens of a workgroup
  int turned; // pieces of a head that turn
  Divisor token_pieces, head_pieces; // (of all of them)
  bool back;
};

struct Turn {
  float cos, sin;
};

// The cosine and sine of position * frequency.  q = 2/pi of the angle's rest
// after n quarter turns is found in 64 bits: the product's own rounding and
// that of 2/pi are added back, so that q is right to 2^-24 of itself for any
// position and frequencies up to 1, or angles up to 2^31.  The series end past
// 2^-28 of their sums at pi/4.
__device__ __forceinline__ Turn turn_of(int position, float frequency) {
  constexpr double kTwoOverPi = 0.63661977236758134308;
  constexpr double kRest = -3.9357353350364972e-17; // 2/pi less that double
  const double p = position, f = frequency;
  const double t = p * f, t_rest = __builtin_fma(p, f, -t);
  const double n = __builtin_rint(t * kTwoOverPi);
  const double q = __builtin_fma(t, kTwoOverPi, -n) +
                   __builtin_fma(t, kRest, t_rest * kTwoOverPi);
  const float r = (float)(q * 1.57079632679489661923);
  const float z = r * r;
  float s = fmaf(z, 1.0f / 362880, -1.0f / 5040);
  s = fmaf(z, s, 1.0f / 120);
  s = fmaf(z, s, -1.0f / 6);
  s = fmaf(r * z, s, r);
  float c = fmaf(z, -1.0f / 3628800, 1.0f / 40320);
  c = fmaf(z, c, -1.0f / 720);
  c = fmaf(z, c, 1.0f / 24);
  c = fmaf(z * z, c, fmaf(z, -0.5f, 1.0f));
  // n modulo 4
  const int turns = (int)(n - 4.0 * __builtin_floor(n * 0.25));
  if (turns & 1) {
    const float x = c;
    c = -s;
    s = x;
  }
  if (turns & 2) {
    c = -c;
    s = -s;
  }
  return {c, s};
}

// W consecutive elements, aligned to one of them, as fp32 and back.  Pieces of 16
// bytes are written past the caches (32,760 tokens of 40 bf16 heads of 128: 110 us,
// 115 with plain stores; 16,384 of 20: 27.1 and 32.8; with loads past them too 107
// and 30.5).
template <typename T, int W> struct Piece {
  typedef T Raw __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  float x[W];
  __device__ __forceinline__ static Raw read(const T *p) {
    return *reinterpret_cast<const Raw *>(p);
  }
  __device__ __forceinline__ static void write(T *p, Raw v) {
    if constexpr (W * sizeof(T) == 16)
      __builtin_nontemporal_store(v, reinterpret_cast<Raw *>(p));
    else
      *reinterpret_cast<Raw *>(p) = v;
  }
  __device__ __forceinline__ void take(Raw v) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      x[i] = tof((T)v[i]);
  }
  __device__ __forceinline__ void load(const T *p) { take(read(p)); }
  __device__ __forceinline__ void store(T *p) const { write(p, raw()); }
  __device__ __forceinline__ Raw raw() const {
    if constexpr (sizeof(T) == 2 && W % 2 == 0) {
      typedef uint32_t Words __attribute__((ext_vector_type(W / 2)));
      Words v;
#pragma unroll
      for (int i = 0; i < W / 2; ++i)
        v[i] = cvt_pk_bf16(x[2 * i], x[2 * i + 1]);
      return __builtin_bit_cast(Raw, v);
    } else if constexpr (sizeof(T) == 2) {
      return Raw{f32_to_bf16(x[0])};
    } else {
      Raw v;
#pragma unroll
      for (int i = 0; i < W; ++i)
        v[i] = x[i];
      return v;
    }
  }
};

__device__ __forceinline__ void turn(float &x, float &y, const Turn &t) {
  const float a = x, b = y;
  x = fmaf(a, t.cos, -(b * t.sin));
  y = fmaf(a, t.sin, b * t.cos);
}

// A head is cut into pieces of W elements.  Of neighbours one holds its pairs, the
// last one maybe with elements that are copied; else two turn with each other, and
// those of the second half start anywhere, as do those that are copied; what is left
// over of either goes in pieces of half the size, a quarter and so on.  (45,248
// tokens of 9 bf16 heads of 96, 25 pairs of neighbours: 26.2 us, in pieces of one
// pair 85.)
template <typename T, int W, bool NEIGHBOURS>
__global__ __launch_bounds__(kThreads) void rotary_turn(RotaryArgs a) {
  extern __shared__ Turn turns[]; // [per][pairs]
  const int first = blockIdx.x * a.per;
  const int count = a.tokens - first < a.per ? a.tokens - first : a.per;
  for (int i = threadIdx.x; i < count * a.pairs; i += kThreads) {
    const int token = i / a.pairs, pair = i - token * a.pairs;
    const int axis = a.axes ? a.axes[pair] : 0;
    Turn t{1.0f, 0.0f}; // (of an axis that is not there)
    if (axis >= 0 && axis < a.axis_count) {
      t = turn_of(a.positions[(int64_t)axis * a.tokens + first + token],
                  a.frequencies[pair]);
      if (a.back)
        t.sin = -t.sin;
    }
    turns[i] = t;
  }
  __syncthreads();
  for (int n = threadIdx.x; n < count * (int)a.token_pieces.by; n += kThreads) {
    const int token = (int)a.token_pieces.quotient(n);
    int u = n - token * (int)a.token_pieces.by;
    int head = (int)a.head_pieces.quotient(u);
    u -= head * (int)a.head_pieces.by;
    const bool key = head >= a.query_heads;
    const Heads &h = key ? a.key : a.query;
    head -= key ? a.query_heads : 0;
    const int64_t at = first + token;
    const T *from = static_cast<const T *>(h.from) + at * h.from_token +
                    head * h.from_head;
    T *to = static_cast<T *>(h.to) + at * h.to_token + head * h.to_head;
    const Turn *t = turns + token * a.pairs;
    const bool copy = u >= a.turned;
    if constexpr (NEIGHBOURS) {
      using P = Piece<T, W>;
      const auto raw = P::read(from + u * W);
      auto out = raw;
      if (!copy) {
        const int some = a.pairs - u * (W / 2); // its pairs
        P p;
        p.take(raw);
#pragma unroll
        for (int e = 0; e < W; e += 2)
          turn(p.x[e], p.x[e + 1],
               t[u * (W / 2) + (e / 2 < some ? e / 2 : 0)]);
        out = p.raw();
        if (some < W / 2)
#pragma unroll
          for (int e = 0; e < W; ++e)
            out[e] = e / 2 < some ? out[e] : raw[e];
      }
      P::write(to + u * W, out);
    } else {
      // N elements of either half, or N that are copied
      auto piece = [&](auto width, int i) __attribute__((always_inline)) {
        constexpr int N = decltype(width)::value;
        Piece<T, N> p, q;
        if (copy) {
          p.write(to + i, p.read(from + i));
          return;
        }
        p.load(from + i);
        q.load(from + i + a.pairs);
#pragma unroll
        for (int e = 0; e < N; ++e)
          turn(p.x[e], q.x[e], t[i + e]);
        p.store(to + i);
        q.store(to + i + a.pairs);
      };
      int i = copy ? 2 * a.pairs + (u - a.turned) * W : u * W;
      const int left = (copy ? a.d : a.pairs) - i;
      if (left >= W) {
        piece(std::integral_constant<int, W>{}, i);
        continue;
      }
      if constexpr (W > 4)
        if (left & 4) {
          piece(std::integral_constant<int, 4>{}, i);
          i += 4;
        }
      if constexpr (W > 2)
        if (left & 2) {
          piece(std::integral_constant<int, 2>{}, i);
          i += 2;
        }
      if (left & 1)
        piece(std::integral_constant<int, 1>{}, i);
    }
  }
}

template <typename T>
int rotary_entry(const int32_t *positions, const float *frequencies,
                 const int32_t *pair_axes, const T *query, const T *key,
                 T *query_output, T *key_output, int64_t tokens, int64_t axes,
                 int64_t query_heads, int64_t key_heads, int64_t d,
                 int64_t pairs, int interleaved, const int64_t *strides,
                 bool back, void *stream) {
  const char *what = back ? "rotary backward" : "rotary";
  sw::clear_error();
  if (tokens < 0 || tokens > sw::kMostTokens || axes < 1 || axes > 65536)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "expected up to 2^30 tokens and 1 to 65536 axes, but got "
                    "%lld and %lld", (long long)tokens, (long long)axes);
  if (query_heads < 1 || query_heads > 65536 || key_heads < 0 ||
      key_heads > 65536)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "expected 1 to 65536 query heads and 0 to 65536 key heads, "
                    "but got %lld and %lld", (long long)query_heads,
                    (long long)key_heads);
  if (d < 8 || d > 128 || d % 8 != 0)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "head dimension must be a multiple of 8 up to 128, but "
                    "got %lld", (long long)d);
  if (pairs < 1 || pairs > d / 2)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "pairs must be 1 to half of the head dimension, but got "
                    "%lld", (long long)pairs);
  if (tokens > 0 && (!positions || !frequencies))
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "%s pointer is null",
                    positions ? "frequencies" : "positions");
  if (int rc = sw::check_value_alignment(4, {positions, frequencies,
                                             pair_axes}))
    return rc;
  const int64_t qs = query_heads * d, ks = key_heads * d;
  const int64_t packed[8] = {qs, d, ks, d, qs, d, ks, d};
  const int64_t *s = strides ? strides : packed;
  const char *names[4] = {"query", "key",
                          back ? "query gradient" : "query output",
                          back ? "key gradient" : "key output"};
  const T *rows[4] = {query, key, query_output, key_output};
  for (int i = 0; i < 4; ++i)
    if (i % 2 == 0 || key_heads > 0)
      if (int rc = check_operand(names[i], rows[i], {s[2 * i], s[2 * i + 1]}, d,
                                 sizeof(T), i >= 2, tokens,
                                 i % 2 ? key_heads : query_heads))
        return rc;
  for (int i = 0; i < 2; ++i)
    if (rows[i] && rows[i] == rows[i + 2] && tokens > 0 &&
        (i == 0 || key_heads > 0) &&
        ((tokens > 1 && s[2 * i] != s[2 * i + 4]) ||
         ((i ? key_heads : query_heads) > 1 && s[2 * i + 1] != s[2 * i + 5])))
      return sw::fail(SW_ERR_INVALID_ARGUMENT,
                      "%s in place needs its input's strides", names[i]);
  if (tokens == 0)
    return SW_OK;
  RotaryArgs a{};
  a.positions = positions;
  a.axes = pair_axes;
  a.frequencies = frequencies;
  a.query = {query, query_output, s[0], s[1], s[4], s[5]};
  a.key = {key, key_output, s[2], s[3], s[6], s[7]};
  a.tokens = (int)tokens;
  a.axis_count = (int)axes;
  a.query_heads = (int)query_heads;
  a.heads = (int)(query_heads + key_heads);
  a.d = (int)d;
  a.pairs = (int)pairs;
  a.back = back;
  // Pieces of 16 bytes, or of 8 where that makes for less work: the pieces, times
  // the rounds of a wave that holds some of what is left over (1, and each smaller
  // size that there is).  (bf16, heads of 40: 59,464 tokens of 5, 20 pairs, 13.9 us
  // and 12.5; 46,588 of 4, 5 pairs, 13.3, with single elements 26; of 80: 16,384 of
  // 20, 10 pairs, 30.6, in twos 37, where the bytes take 16.6: pairs that are no
  // whole pieces, whose second halves start off their alignment, cost that much.)
  constexpr int kWide = 16 / sizeof(T);
  const int64_t copied = d - 2 * pairs;
  auto pieces = [&](int64_t w) {
    return sw::ceil_div(pairs, w) + sw::ceil_div(copied, w);
  };
  auto work = [&](int64_t w) {
    const int64_t rest = pairs % w | copied % w;
    return pieces(w) * (1 + (rest & 1) + (rest >> 1 & 1) + (rest >> 2));
  };
  const bool narrow = !interleaved && work(kWide / 2) < work(kWide);
  const int64_t width = narrow ? kWide / 2 : kWide;
  const int64_t all = interleaved ? d / width : pieces(width);
  a.turned = (int)sw::ceil_div((interleaved ? 2 : 1) * pairs, width);
  a.head_pieces = Divisor((uint32_t)all);
  a.token_pieces = Divisor((uint32_t)(all * a.heads));
  // (two pieces a thread; with four 16,384 and 32,760 tokens take 4 to 10 % longer)
  a.per = (int)std::clamp<int64_t>(2 * kThreads / (all * a.heads), 1, 16);
  const int64_t grid = sw::ceil_div(tokens, a.per);
  if (int rc = sw::check_flat_grid(grid, kThreads, what))
    return rc;
  const hipStream_t st = sw::as_stream(stream);
  const dim3 g((unsigned)grid);
  const size_t lds = a.per * a.pairs * sizeof(Turn);
  if (interleaved)
    rotary_turn<T, kWide, true><<<g, kThreads, lds, st>>>(a);
  else if (narrow)
    rotary_turn<T, kWide / 2, false><<<g, kThreads, lds, st>>>(a);
  else
    rotary_turn<T, kWide, false><<<g, kThreads, lds, st>>>(a);
  return sw::launch_check(what);
}

} // namespace

extern "C" int sw_rotary_f32(
    const int32_t *positions, const float *frequencies,
    const int32_t *pair_axes, const float *query, const float *key,
    float *query_output, float *key_output, int64_t tokens, int64_t axes,
    int64_t query_heads, int64_t key_heads, int64_t d, int64_t pairs,
    int interleaved, const int64_t *strides, void *stream) {
  return rotary_entry<float>(positions, frequencies, pair_axes, query, key,
                             query_output, key_output, tokens, axes,
                             query_heads, key_heads, d, pairs, interleaved,
                             strides, false, stream);
}

extern "C" int sw_rotary_bf16(
    const int32_t *positions, const float *frequencies,
    const int32_t *pair_axes, const uint16_t *query, const uint16_t *key,
    uint16_t *query_output, uint16_t *key_output, int64_t tokens, int64_t axes,
    int64_t query_heads, int64_t key_heads, int64_t d, int64_t pairs,
    int interleaved, const int64_t *strides, void *stream) {
  return rotary_entry<uint16_t>(positions, frequencies, pair_axes, query, key,
                                query_output, key_output, tokens, axes,
                                query_heads, key_heads, d, pairs, interleaved,
                                strides, false, stream);
}

extern "C" int sw_rotary_backward_f32(
    const int32_t *positions, const float *frequencies,
    const int32_t *pair_axes, const float *query_output_gradient,
    const float *key_output_gradient, float *query_gradient,
    float *key_gradient, int64_t tokens, int64_t axes, int64_t query_heads,
    int64_t key_heads, int64_t d, int64_t pairs, int interleaved,
    const int64_t *strides, void *stream) {
  return rotary_entry<float>(positions, frequencies, pair_axes,
                             query_output_gradient, key_output_gradient,
                             query_gradient, key_gradient, tokens, axes,
                             query_heads, key_heads, d, pairs, interleaved,
                             strides, true, stream);
}

extern "C" int sw_rotary_backward_bf16(
    const int32_t *positions, const float *frequencies,
    const int32_t *pair_axes, const uint16_t *query_output_gradient,
    const uint16_t *key_output_gradient, uint16_t *query_gradient,
    uint16_t *key_gradient, int64_t tokens, int64_t axes, int64_t query_heads,
    int64_t key_heads, int64_t d, int64_t pairs, int interleaved,
    const int64_t *strides, void *stream) {
  return rotary_entry<uint16_t>(positions, frequencies, pair_axes,
                                query_output_gradient, key_output_gradient,
                                query_gradient, key_gradient, tokens, axes,
                                query_heads, key_heads, d, pairs, interleaved,
                                strides, true, stream);
}
