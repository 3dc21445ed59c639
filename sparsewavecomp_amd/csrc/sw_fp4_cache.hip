// Keys and values into a cache of 4-bit codes, and back: packed tokens of
// sequences whose places lie in pages (sw_fp4.h has the rows' format).
//
// Both directions move each element once, two to four bytes of it on one side
// and 17/32 on the other, and compute little: memory bounds them, and for few
// tokens the chain of reads that leads to a token's page (offsets, length,
// table).  32,768 tokens of 8 heads of 128, bf16: written in 36 us, 4.7 TB/s, read
// back in 29, 5.9 TB/s; a large copy reaches 6.3.  One token of each of 64 sequences:
// 4.4 and 4.0 us.
#include "sw_fp4.h"
#include "sw_internal.h"

#include <type_traits>

using namespace swd;
using sw::check_operand;

namespace {

constexpr int kThreads = 256;
// elements of a lane, 16 bytes of them: a block lies in 32 / kUnit lanes
template <typename T> constexpr int kUnit = 16 / (int)sizeof(T);

struct Rows {
  uint8_t *codes, *scales;
  int64_t codes_page, codes_token, codes_head; // strides in bytes
  int64_t scales_page, scales_token, scales_head;
};

struct MoveArgs {
  // write: `from` holds the lengths of the sequences' keys, whose last ones
  // the tokens are; read: the place of the first token (null: 0)
  const int32_t *offsets, *from, *table;
  void *key, *value;
  int64_t key_token, key_head, value_token, value_head;
  Rows keys, values;
  int sequences, tokens, pages, table_width, heads;
  int64_t room; // places of a sequence
  int at_once; // tokens that a wave moves at once, 64 / lanes
  Divisor page_size, lanes, rows; // lanes of a token; rows: 2 heads
};

constexpr int kNoPage = -1, kNoSequence = -2; // in the place of `codes`
struct Place {
  int64_t codes, scales; // where a head's row starts, from its first row on
};

// Lane l: the place of token first + l (first is wave-uniform) in a cache's keys
// or values.
template <bool WRITE>
__device__ __forceinline__ Place place_of(const MoveArgs &a, const Rows &rows,
                                          int first, bool live) {
  const int l = lane_id(), token = first + l, n = a.sequences;
  const int32_t *offsets = a.offsets;
  const int base =
      n <= kWave ? 0
                 : last_at_most(n, first, [&](int i) { return offsets[i]; });
  // how many of the next 64 sequences end at or before the token
  const int end_of = base + l < n ? offsets[base + l + 1] : INT32_MAX;
  int i = 0;
#pragma unroll
  for (int step = 32; step > 0; step >>= 1)
    if (__builtin_amdgcn_ds_bpermute((i + step - 1) * 4, end_of) <= token)
      i += step;
  i += base;
  if (i == base + 63) { // (or more: a search of the rest)
    int to = n;
    while (i < to) {
      const int mid = i + (to - i) / 2;
      if (offsets[mid + 1] <= token)
        i = mid + 1;
      else
        to = mid;
    }
  }
  Place p{kNoSequence, 0};
  if (!live || i >= n)
    return p;
  const int64_t begin = offsets[i], end = offsets[i + 1];
  if (token < begin || token >= end)
    return p;
  const int64_t place = WRITE ? a.from[i] - (end - token)
                              : (a.from ? a.from[i] : 0) + (token - begin);
  p.codes = kNoPage;
  if (place < 0 || place >= a.room)
    return p;
  const int number = (int)a.page_size.quotient((uint32_t)place);
  const int64_t page =
      a.table ? a.table[(int64_t)i * a.table_width + number] : i;
  if (page < 0 || page >= a.pages)
    return p;
  const int64_t slot = (int)place - number * (int)a.page_size.by;
  p.codes = page * rows.codes_page + slot * rows.codes_token;
  p.scales = page * rows.scales_page + slot * rows.scales_token;
  return p;
}
// What `lane` holds in v.
__device__ __forceinline__ int64_t of_lane(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(lane * 4, (int)v);
  const int hi = __builtin_amdgcn_ds_bpermute(lane * 4, (int)(v >> 32));
  return (int64_t)hi << 32 | lo;
}

// What a wave moves: the keys or the values of one head, of PASSES times
// `at_once` consecutive tokens.  Their codes lie next to each other in a page that
// holds a head's rows together, their scales too, so that lines are written whole;
// of the tokens' side 16 bytes a lane are whole lines in any case.  (A token's keys
// and values of all heads in a workgroup: 134 MB written 54.8 us, read 53; 600 MB
// read 216.)
template <typename T> struct Wave {
  bool value, any;
  int first, token, piece; // the wave's first token; this lane's of a pass
  int64_t token_stride, at; // of a lane's elements
  const Rows &rows;
  uint8_t *codes, *scales; // of this lane in the head's first row
  __device__ __forceinline__ Wave(const MoveArgs &a, int passes, int number,
                                  int tile)
      : value(number - tile * (int)a.rows.by >= a.heads),
        rows(value ? a.values : a.keys) {
    const int head = number - tile * (int)a.rows.by - (value ? a.heads : 0);
    first = tile * passes * a.at_once;
    any = first < a.tokens;
    token = (int)a.lanes.quotient(lane_id());
    piece = lane_id() - token * (int)a.lanes.by;
    token_stride = value ? a.value_token : a.key_token;
    at = head * (value ? a.value_head : a.key_head) + piece * kUnit<T>;
    codes = rows.codes + head * rows.codes_head + piece * (kUnit<T> / 2);
    scales = rows.scales + head * rows.scales_head + piece * kUnit<T> / 32;
  }
};
template <typename T>
__device__ __forceinline__ Wave<T> wave_of(const MoveArgs &a, int passes) {
  const int number = (int)blockIdx.x * (kThreads / kWave) + wave_in_group();
  return {a, passes, number, (int)a.rows.quotient(number)};
}

// Units pass by the caches.  Reads of the tokens' side: written 32,768 tokens of
// 8 heads of 128, bf16, 38 us, 44 with plain loads.  Writes of it: read back
// 28.8 us with them, 38.9 plain; 262,144 tokens at most of 4 sequences 133 and 145;
// in fp32 53 and 83.  A kernel that reads 67 to 134 MB of them right away finds
// less in the caches (sum of both: 72 us against 68, 39 and 36), of smaller and
// larger ones or in fp32 the sum is smaller too (13 and 13.6, 291 and 299, 150 and
// 164).
__device__ __forceinline__ v4u load_unit(const void *p) {
  return __builtin_nontemporal_load(static_cast<const v4u *>(p));
}
__device__ __forceinline__ void store_unit(void *p, v4u x) {
  __builtin_nontemporal_store(x, static_cast<v4u *>(p));
}

// Of the block that a lane's unit lies in, the largest size's bits.
__device__ __forceinline__ uint32_t block_top(v4u x, uint16_t) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = max(top, max(x[i] & 0x7FFF0000u, x[i] << 16 & 0x7FFF0000u));
  top = max(top, (uint32_t)dpp_i<kQuadXor1>(0, (int)top));
  return max(top, (uint32_t)dpp_i<kQuadXor2>(0, (int)top));
}
__device__ __forceinline__ uint32_t block_top(v4u x, float) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = max(top, x[i] & 0x7FFFFFFFu);
  top = max(top, (uint32_t)dpp_i<kQuadXor1>(0, (int)top));
  top = max(top, (uint32_t)dpp_i<kQuadXor2>(0, (int)top));
  return max(top, (uint32_t)dpp_i<kRowHalfMirror>(0, (int)top));
}

// The codes of a unit: four bytes of bf16 values, two of fp32 ones.
template <typename T> struct Codes;
template <> struct Codes<uint16_t> {
  using Word = uint32_t;
  __device__ static __forceinline__ Word of(v4u x, float scale) {
    return fp4_codes(x, scale);
  }
  __device__ static __forceinline__ v4u values(Word codes, float scale) {
    return fp4_values(codes, scale);
  }
};
template <> struct Codes<float> {
  using Word = uint16_t;
  __device__ static __forceinline__ Word of(v4u x, float scale) {
    return (Word)fp4_codes(__builtin_bit_cast(v4f, x), scale);
  }
  __device__ static __forceinline__ v4u values(Word codes, float scale) {
    return fp4_values_f32(codes, scale);
  }
};

template <typename T, int PASSES>
__global__ __launch_bounds__(kThreads) void fp4_cache_write(MoveArgs a) {
  using C = Codes<T>;
  const Wave<T> w = wave_of<T>(a, PASSES);
  if (!w.any)
    return;
  const T *from = static_cast<const T *>(w.value ? a.value : a.key) + w.at;
  const bool lane = w.token < a.at_once; // (some are left over of rows of 96)
  v4u x[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int token = w.first + i * a.at_once + w.token;
    x[i] = v4u{};
    if (lane && token < a.tokens)
      x[i] = load_unit(from + token * w.token_stride);
  }
  const Place all = place_of<true>(a, w.rows, w.first,
                                   lane_id() < PASSES * a.at_once &&
                                       w.first + lane_id() < a.tokens);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int of = i * a.at_once + w.token;
    const int64_t at = of_lane(all.codes, of), scale = of_lane(all.scales, of);
    const uint32_t byte = fp4_scale_byte(block_top(x[i], T{}));
    const typename C::Word codes =
        byte == 255 ? 0u : C::of(x[i], fp4_scale(byte));
    if (lane && at >= 0) {
      *reinterpret_cast<typename C::Word *>(w.codes + at) = codes;
      if (w.piece % (32 / kUnit<T>) == 0)
        w.scales[scale] = (uint8_t)byte;
    }
  }
}

template <typename T, int PASSES>
__global__ __launch_bounds__(kThreads) void fp4_cache_read(MoveArgs a) {
  using C = Codes<T>;
  const Wave<T> w = wave_of<T>(a, PASSES);
  if (!w.any)
    return;
  const bool lane = w.token < a.at_once;
  const Place all = place_of<false>(a, w.rows, w.first,
                                    lane_id() < PASSES * a.at_once &&
                                        w.first + lane_id() < a.tokens);
  int state[PASSES];
  typename C::Word codes[PASSES];
  uint8_t bytes[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int of = i * a.at_once + w.token;
    const int64_t at = of_lane(all.codes, of), scale = of_lane(all.scales, of);
    state[i] = (int)(at >> 32) < 0 ? (int)at : 0;
    codes[i] = 0;
    bytes[i] = 0;
    if (lane && at >= 0) {
      codes[i] = *reinterpret_cast<const typename C::Word *>(w.codes + at);
      bytes[i] = w.scales[scale];
    }
  }
  T *to = static_cast<T *>(w.value ? a.value : a.key) + w.at;
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
    if (lane && state[i] != kNoSequence)
      store_unit(to + (w.first + i * a.at_once + w.token) * w.token_stride,
                 C::values(codes[i], fp4_scale(bytes[i])));
}

// ---- host ------------------------------------------------------------------------

template <bool WRITE, typename T>
int move_entry(const int32_t *token_offsets, const int32_t *from,
               const int32_t *page_table, const T *key, const T *value,
               const uint8_t *key_codes, const uint8_t *key_scales,
               const uint8_t *value_codes, const uint8_t *value_scales,
               int64_t sequences, int64_t tokens, int64_t pages,
               int64_t page_size, int64_t table_width, int64_t key_heads,
               int64_t d, const int64_t *strides, void *stream) {
  const char *what = WRITE ? "fp4 cache write" : "fp4 cache read";
  sw::clear_error();
  if (!page_table)
    table_width = 1;
  if (int rc = sw::check_cache_sizes(sequences, tokens, pages, page_size,
                                     table_width, page_table != nullptr))
    return rc;
  if (int rc = sw::check_fp4_heads(key_heads, key_heads, d))
    return rc;
  if (sequences > 0 && tokens > 0 && !token_offsets)
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "token offsets pointer is null");
  if (WRITE && sequences > 0 && tokens > 0 && !from)
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "key lengths pointer is null");
  if (int rc = sw::check_value_alignment(4, {token_offsets, from, page_table}))
    return rc;
  int64_t packed[16];
  sw::fp4_packed_strides(packed, key_heads, key_heads, page_size, d);
  const int64_t *s = strides ? strides : packed;
  const char *names[2] = {"key", "value"};
  const T *rows[2] = {key, value};
  for (int i = 0; i < 2; ++i)
    if (int rc = check_operand(names[i], rows[i], {s[2 * i], s[2 * i + 1]}, d,
                               sizeof(T), !WRITE, tokens, key_heads))
      return rc;
  if (int rc = sw::check_fp4_cache("key", key_codes, key_scales, s + 4, d,
                                   pages, page_size, key_heads, WRITE))
    return rc;
  if (int rc = sw::check_fp4_cache("value", value_codes, value_scales, s + 10,
                                   d, pages, page_size, key_heads, WRITE))
    return rc;
  if (sequences == 0 || tokens == 0)
    return SW_OK;
  MoveArgs a{};
  a.offsets = token_offsets;
  a.from = from;
  a.table = page_table;
  a.key = const_cast<T *>(key);
  a.value = const_cast<T *>(value);
  a.key_token = s[0];
  a.key_head = s[1];
  a.value_token = s[2];
  a.value_head = s[3];
  a.keys = {const_cast<uint8_t *>(key_codes), const_cast<uint8_t *>(key_scales),
            s[4], s[5], s[6], s[7], s[8], s[9]};
  a.values = {const_cast<uint8_t *>(value_codes),
              const_cast<uint8_t *>(value_scales),
              s[10], s[11], s[12], s[13], s[14], s[15]};
  a.sequences = (int)sequences;
  a.tokens = (int)tokens;
  a.pages = (int)pages;
  a.table_width = (int)table_width;
  a.room = page_size * table_width;
  a.page_size = Divisor((uint32_t)page_size);
  a.heads = (int)key_heads;
  a.lanes = Divisor((uint32_t)(d / kUnit<T>));
  a.rows = Divisor((uint32_t)(2 * key_heads));
  a.at_once = (int)(kWave / (d / kUnit<T>));
  const int64_t bytes = 2 * tokens * key_heads * d * (int64_t)sizeof(T);
  // Passes of a wave, us (keys and values in bytes; write, read back):
  //            0.26 MB     4.2 MB      6.9 MB (fp32)  16.8 MB     67 MB        134 MB       600 MB
  //   1        3.5, 3.3    4.2, 4.0    6.7, 5.5       10.5, 8.8   31.0, 25.3   57.0, 46.3   -, 265
  //   4        4.5, 4.2    4.8, 4.5    5.7, 4.9        8.6, 6.9   23.0, 16.5   39.9, 27.8   -, 162
  //   8        5.7, 5.4    6.1, 5.6    6.7, 6.0        8.9, 7.1   21.4, 16.4   37.8, 28.7   -, 132
  // (and 64 tokens at most, whose places a wave finds at once)
  int64_t passes = bytes < (6 << 20) ? 1 : bytes < (48 << 20) ? 4 : 8;
  if (passes * a.at_once > kWave)
    passes = 4;
  const int64_t waves =
      sw::ceil_div(tokens, a.at_once * passes) * 2 * key_heads;
  const int64_t grid = sw::ceil_div(waves, kThreads / kWave);
  if (waves > INT32_MAX)
    return sw::fail(SW_ERR_INVALID_SHAPE, "%s of %lld tokens and %lld heads is "
                    "more than one launch holds", what, (long long)tokens,
                    (long long)key_heads);
  if (int rc = sw::check_flat_grid(grid, kThreads, what))
    return rc;
  const hipStream_t st = sw::as_stream(stream);
  const dim3 g((unsigned)grid);
  auto launch = [&](auto count) {
    constexpr int N = decltype(count)::value;
    if constexpr (WRITE)
      fp4_cache_write<T, N><<<g, kThreads, 0, st>>>(a);
    else
      fp4_cache_read<T, N><<<g, kThreads, 0, st>>>(a);
  };
  if (passes == 1)
    launch(std::integral_constant<int, 1>{});
  else if (passes == 4)
    launch(std::integral_constant<int, 4>{});
  else
    launch(std::integral_constant<int, 8>{});
  return sw::launch_check(what);
}

} // namespace

extern "C" int sw_fp4_cache_write_f32(
    const int32_t *token_offsets, const int32_t *key_lengths,
    const int32_t *page_table, const float *key, const float *value,
    uint8_t *key_codes, uint8_t *key_scales, uint8_t *value_codes,
    uint8_t *value_scales, int64_t sequences, int64_t tokens, int64_t pages,
    int64_t page_size, int64_t table_width, int64_t key_heads, int64_t d,
    const int64_t *strides, void *stream) {
  return move_entry<true, float>(
      token_offsets, key_lengths, page_table, key, value, key_codes, key_scales,
      value_codes, value_scales, sequences, tokens, pages, page_size,
      table_width, key_heads, d, strides, stream);
}

extern "C" int sw_fp4_cache_write_bf16(
    const int32_t *token_offsets, const int32_t *key_lengths,
    const int32_t *page_table, const uint16_t *key, const uint16_t *value,
    uint8_t *key_codes, uint8_t *key_scales, uint8_t *value_codes,
    uint8_t *value_scales, int64_t sequences, int64_t tokens, int64_t pages,
    int64_t page_size, int64_t table_width, int64_t key_heads, int64_t d,
    const int64_t *strides, void *stream) {
  return move_entry<true, uint16_t>(
      token_offsets, key_lengths, page_table, key, value, key_codes, key_scales,
      value_codes, value_scales, sequences, tokens, pages, page_size,
      table_width, key_heads, d, strides, stream);
}

extern "C" int sw_fp4_cache_read_f32(
    const int32_t *token_offsets, const int32_t *starts,
    const int32_t *page_table, const uint8_t *key_codes,
    const uint8_t *key_scales, const uint8_t *value_codes,
    const uint8_t *value_scales, float *key, float *value, int64_t sequences,
    int64_t tokens, int64_t pages, int64_t page_size, int64_t table_width,
    int64_t key_heads, int64_t d, const int64_t *strides, void *stream) {
  return move_entry<false, float>(
      token_offsets, starts, page_table, key, value, key_codes, key_scales,
      value_codes, value_scales, sequences, tokens, pages, page_size,
      table_width, key_heads, d, strides, stream);
}

extern "C" int sw_fp4_cache_read_bf16(
    const int32_t *token_offsets, const int32_t *starts,
    const int32_t *page_table, const uint8_t *key_codes,
    const uint8_t *key_scales, const uint8_t *value_codes,
    const uint8_t *value_scales, uint16_t *key, uint16_t *value,
    int64_t sequences, int64_t tokens, int64_t pages, int64_t page_size,
    int64_t table_width, int64_t key_heads, int64_t d, const int64_t *strides,
    void *stream) {
  return move_entry<false, uint16_t>(
      token_offsets, starts, page_table, key, value, key_codes, key_scales,
      value_codes, value_scales, sequences, tokens, pages, page_size,
      table_width, key_heads, d, strides, stream);
}
