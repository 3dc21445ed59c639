// Keys and values into a cache of 4-bit codes, and back: packed tokens of
// sequences whose places lie in pages (sw_fp4.h has the rows' format).
//
// Both directions move each element once, two to four bytes of it on one side
// and 17/32 on the other, and compute little: memory bounds them, and for few
// tokens the chain of reads that leads to a token's page (offsets, length,
// table).
#include "sw_fp4.h"
#include "sw_internal.h"

#include <algorithm>

using namespace swd;
using sw::check_operand;

namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8; // elements of a thread: four threads hold a block

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
  int sequences, tokens, pages, table_width, units;
  int64_t room; // places of a sequence
  int team; // log2 of the threads that share a token
  Divisor page_size, row_units;
};

constexpr int kNoPage = -1, kNoSequence = -2;
struct Place {
  int page, slot;
};

// Lane l: the place of token first + l (first is wave-uniform).
template <bool WRITE>
__device__ __forceinline__ Place place_of(const MoveArgs &a, int first,
                                          bool live) {
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
  p.page = kNoPage;
  if (place < 0 || place >= a.room)
    return p;
  const int number = (int)a.page_size.quotient((uint32_t)place);
  const int page =
      a.table ? a.table[(int64_t)i * a.table_width + number] : i;
  if (page < 0 || page >= a.pages)
    return p;
  p.page = page;
  p.slot = (int)place - number * (int)a.page_size.by;
  return p;
}

// Which elements a thread takes of a token: unit `u` of those of its keys and
// then of its values.
struct Unit {
  bool value;
  int head, piece;
  __device__ __forceinline__ Unit(const MoveArgs &a, int u) {
    value = 2 * u >= a.units;
    u -= value ? a.units / 2 : 0;
    head = (int)a.row_units.quotient(u);
    piece = u - head * (int)a.row_units.by;
  }
  __device__ __forceinline__ int64_t element(const MoveArgs &a,
                                             int token) const {
    return token * (value ? a.value_token : a.key_token) +
           head * (value ? a.value_head : a.key_head) + piece * kUnit;
  }
  __device__ __forceinline__ uint32_t *codes(const MoveArgs &a,
                                             const Place &p) const {
    const Rows &r = value ? a.values : a.keys;
    return reinterpret_cast<uint32_t *>(
        r.codes + p.page * r.codes_page + p.slot * r.codes_token +
        head * r.codes_head + piece * 4);
  }
  __device__ __forceinline__ uint8_t *scale(const MoveArgs &a,
                                            const Place &p) const {
    const Rows &r = value ? a.values : a.keys;
    return r.scales + p.page * r.scales_page + p.slot * r.scales_token +
           head * r.scales_head + piece / 4;
  }
};

// A workgroup takes PER tokens for each of its teams of 2^team threads, team t
// the tokens t, t + teams, ...; a wave finds the places of them all, one a lane.
template <typename T, int PER>
__global__ __launch_bounds__(kThreads) void fp4_cache_write(MoveArgs a) {
  const int team = threadIdx.x >> a.team, teams = kThreads >> a.team;
  const int first = blockIdx.x * teams * PER;
  int u = threadIdx.x & ((1 << a.team) - 1);
  Frag<T> x[PER];
  auto load = [&]() __attribute__((always_inline)) {
    const Unit unit(a, u);
    const T *from = static_cast<const T *>(unit.value ? a.value : a.key);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int token = first + i * teams + team;
      x[i] = token < a.tokens ? ld_frag(from + unit.element(a, token))
                              : zero_frag<T>();
    }
  };
  if (u < a.units)
    load();
  const Place all = place_of<true>(
      a, first, lane_id() < teams * PER && first + lane_id() < a.tokens);
  Place p[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int from = (i * teams + team) * 4;
    p[i].page = __builtin_amdgcn_ds_bpermute(from, all.page);
    p[i].slot = __builtin_amdgcn_ds_bpermute(from, all.slot);
  }
  while (u < a.units) {
    const Unit unit(a, u);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      // (a block lies in four neighbours, all of one team)
      int top = (int)top_bits(x[i]);
      top = max(top, dpp_i<kQuadXor1>(0, top));
      top = max(top, dpp_i<kQuadXor2>(0, top));
      const uint32_t byte = fp4_scale_byte((uint32_t)top);
      const uint32_t codes =
          byte == 255 ? 0u : fp4_codes(x[i], fp4_scale(byte));
      if (p[i].page >= 0) {
        *unit.codes(a, p[i]) = codes;
        if (unit.piece % 4 == 0)
          *unit.scale(a, p[i]) = (uint8_t)byte;
      }
    }
    u += 1 << a.team;
    if (u < a.units)
      load();
  }
}

__device__ __forceinline__ void store_values(uint16_t *p, uint32_t codes,
                                             float scale) {
  *reinterpret_cast<v4u *>(p) = fp4_values(codes, scale);
}
__device__ __forceinline__ void store_values(float *p, uint32_t codes,
                                             float scale) {
  const v4u x = fp4_values(codes, scale);
#pragma unroll
  for (int i = 0; i < 4; i += 2)
    *reinterpret_cast<v4f *>(p + 2 * i) =
        v4f{__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xFFFF0000u),
            __uint_as_float(x[i + 1] << 16),
            __uint_as_float(x[i + 1] & 0xFFFF0000u)};
}

template <typename T, int PER>
__global__ __launch_bounds__(kThreads) void fp4_cache_read(MoveArgs a) {
  const int team = threadIdx.x >> a.team, teams = kThreads >> a.team;
  const int first = blockIdx.x * teams * PER;
  const Place all = place_of<false>(
      a, first, lane_id() < teams * PER && first + lane_id() < a.tokens);
  Place p[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int from = (i * teams + team) * 4;
    p[i].page = __builtin_amdgcn_ds_bpermute(from, all.page);
    p[i].slot = __builtin_amdgcn_ds_bpermute(from, all.slot);
  }
  for (int u = threadIdx.x & ((1 << a.team) - 1); u < a.units;
       u += 1 << a.team) {
    const Unit unit(a, u);
    T *to = static_cast<T *>(unit.value ? a.value : a.key);
    uint32_t codes[PER], bytes[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      codes[i] = p[i].page >= 0 ? *unit.codes(a, p[i]) : 0u;
      bytes[i] = p[i].page >= 0 ? *unit.scale(a, p[i]) : 0u;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (p[i].page != kNoSequence)
        store_values(to + unit.element(a, first + i * teams + team), codes[i],
                     fp4_scale(bytes[i]));
  }
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
  a.row_units = Divisor((uint32_t)(d / kUnit));
  a.units = (int)(2 * key_heads * (d / kUnit));
  a.team = 2;
  while (a.team < 8 && 1 << a.team < a.units)
    ++a.team;
  const int64_t teams = kThreads >> a.team;
  const int64_t per = tokens >= 4096 * teams && teams <= 16 ? 4 : 1;
  const int64_t grid = sw::ceil_div(tokens, teams * per);
  if (int rc = sw::check_flat_grid(grid, kThreads, what))
    return rc;
  const hipStream_t st = sw::as_stream(stream);
  const dim3 g((unsigned)grid);
  if (WRITE && per == 4)
    fp4_cache_write<T, 4><<<g, kThreads, 0, st>>>(a);
  else if (WRITE)
    fp4_cache_write<T, 1><<<g, kThreads, 0, st>>>(a);
  else if (per == 4)
    fp4_cache_read<T, 4><<<g, kThreads, 0, st>>>(a);
  else
    fp4_cache_read<T, 1><<<g, kThreads, 0, st>>>(a);
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
