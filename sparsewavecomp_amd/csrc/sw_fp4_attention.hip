// Attention of one query for each sequence against a key-value cache of 4-bit
// codes, over a sliding window with sinks.
//
// The arithmetic of the cache attention over bf16 values (sw_cache_attention.hip):
// a code times its block's scale is a bf16 number, so the bf16 matrix cores
// multiply with it exactly, and fp32 queries, cut into three bf16 parts, and
// probabilities lose nothing either.  A key and its value take 17/16 d bytes for
// 4 G d operations of the G query heads that share them: 3.75 times fewer bytes
// than in bf16, for the same products, exponentials and conversions besides.
#include "sw_cache.h"
#include "sw_fp4.h"

namespace {

struct Scales {
  const uint8_t *key, *value;
  int64_t key_page, key_token, key_head; // strides in bytes
  int64_t value_page, value_token, value_head;
};

struct Fp4StepArgs {
  StepArgs s; // (its cache: the codes, strides in bytes)
  Scales scales;
  Divisor page_size;
};

// bf16 parts of a query's elements and of a probability: of fp32 operands all 24
// bits.  bf16 probabilities keep 15 bits, as in the attention of bf16 caches.
template <typename T> constexpr int kQueryParts = sizeof(T) == 4 ? 3 : 1;
template <typename T> constexpr int kWeightParts = sizeof(T) == 4 ? 3 : 2;

// Eight elements as fragments of bf16 whose sum they are.  What is left of an
// element that is not zero is at least 2^-126, so that an infinity of a key (code
// times a scale that passes fp32's range) meets no zero; that moves elements of
// 2^-100 and more by 2^-25 of themselves at most, smaller ones by no more.
__device__ __forceinline__ void query_parts(v4u x, v4u (&part)[1]) {
  part[0] = x;
}
__device__ __forceinline__ void query_parts(v8f x, v4u (&part)[3]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    r[e] = x[e];
#pragma unroll
  for (int p = 0; p < 3; ++p) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      part[p][e] = __builtin_amdgcn_perm(__float_as_uint(r[2 * e + 1]),
                                         __float_as_uint(r[2 * e]), 0x07060302u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float rest =
          r[e] - __uint_as_float(__float_as_uint(r[e]) & 0xFFFF0000u);
      r[e] = copysignf(
          fmaxf(fabsf(rest), fminf(fabsf(x[e]) * 0x1p-26f, 0x1p-126f)), x[e]);
    }
  }
}

// Eight probabilities as two fragments to 2^-15, or three to 2^-23 of each (as
// split_frag: what is left of one is at least 2^-126).
__device__ __forceinline__ void weight_parts(const float *x, v4u (&part)[2]) {
  split_frag(x, part[0], part[1]);
}
__device__ __forceinline__ void weight_parts(const float *x, v4u (&part)[3]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    r[e] = __builtin_amdgcn_fmed3f(
        x[e] - __uint_as_float(__float_as_uint(x[e]) & 0xFFFF0000u), 0x1p-126f,
        x[e]);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    part[0][e] = __builtin_amdgcn_perm(__float_as_uint(x[2 * e + 1]),
                                       __float_as_uint(x[2 * e]), 0x07060302u);
  split_frag(r, part[1], part[2]);
}

// One chunk of keys against up to 16 query rows, 32 keys a wave at a time: lane
// l holds a quarter (l / 16) of the keys l % 16 and 16 + l % 16, whose codes are
// one load for d = 128; quarter g of step st is elements D / 4 g + 8 st + i of
// the products' K index, in the queries too.  Values go through LDS as bf16, to
// be read across their rows.
template <typename T, int D> struct Fp4Parts {
  using Tile = RowTile<uint16_t, D, kTile, kWave>;
  static constexpr int kWaveBytes =
      Tile::kBytes > kRows * D * 4 ? Tile::kBytes : kRows * D * 4;
  static constexpr int kBytes = 4 * kWaveBytes;
  static constexpr int kWaves = sizeof(T) == 4 ? 2 : D > 64 ? 3 : 4;
};

template <typename T, int D>
__global__ __launch_bounds__(kThreads, (Fp4Parts<T, D>::kWaves)) void
fp4_cache_parts(Fp4StepArgs args) {
  using Tile = typename Fp4Parts<T, D>::Tile;
  constexpr int kSteps = D / 32;  // products along d
  constexpr int kBlocks = D / 16; // output rows of 16
  constexpr int kWords = D / 32;  // words of codes of a lane's quarter row
  constexpr int kWaveBytes = Fp4Parts<T, D>::kWaveBytes;
  __shared__ __align__(1024) char lds[Fp4Parts<T, D>::kBytes];
  __shared__ Totals found;
  const StepArgs &a = args.s;

  const int lane = lane_id(), g = lane >> 4, wave = wave_in_group();
  int64_t item = blockIdx.x;
  const int part = (int)(item % a.parts);
  item /= a.parts;
  const int first_row = (int)(item % (a.rows / kRows)) * kRows;
  item /= a.rows / kRows;
  const int hk = (int)(item % a.key_heads);
  const int seq = (int)(item / a.key_heads);
  const Visible see(a, seq);
  const int v0 = part * a.chunk;
  const int v1 = see.count < v0 + a.chunk ? see.count : v0 + a.chunk;
  const int64_t of =
      (((int64_t)seq * a.key_heads + hk) * a.parts + part) * a.rows + first_row;
  const bool only = a.parts == 1;
  if (v1 <= v0 && !only)
    return;
  const int rows = a.group - first_row < kRows ? a.group - first_row : kRows;

  const bool none = a.alpha == 0.0f;
  const float scale = none ? 1.0f : fabsf(a.alpha) * kLog2e;
  const bool live = (lane & 15) < rows;
  v4u q[kQueryParts<T>][kSteps];
  {
    const int row = first_row + (live ? lane & 15 : 0);
    const T *p = static_cast<const T *>(a.query) + seq * a.query_token +
                 (hk * a.group + row) * a.query_head;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int c = D / 4 * g + 8 * st;
      Frag<T> x = live && c < a.d && !none ? ld_frag(p + c) : zero_frag<T>();
      if (a.alpha < 0.0f)
        x = negate_frag<T>(x);
      v4u cut[kQueryParts<T>];
      query_parts(x, cut);
#pragma unroll
      for (int i = 0; i < kQueryParts<T>; ++i)
        q[i][st] = cut[i];
    }
  }

  // this lane's quarter of a row: codes, and the scale of its block
  const int code_at = D / 8 * g, scale_at = D * g / 128;
  const bool inside = code_at * 2 < a.d;
  const uint8_t *zeros = reinterpret_cast<const uint8_t *>(kZeros);
  const uint8_t *key_codes = static_cast<const uint8_t *>(a.cache.key) +
                             hk * a.cache.key_head + code_at;
  const uint8_t *value_codes = static_cast<const uint8_t *>(a.cache.value) +
                               hk * a.cache.value_head + code_at;
  const uint8_t *key_scales =
      args.scales.key + hk * args.scales.key_head + scale_at;
  const uint8_t *value_scales =
      args.scales.value + hk * args.scales.value_head + scale_at;
  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  struct Data {
    Words key[2], value[2];
    uint32_t key_scale[2], value_scale[2];
    uint32_t none; // bit i: key i of this lane's scores is none
  };
  auto fetch = [&](int v) __attribute__((always_inline)) {
    Data x;
    uint64_t has[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int at = v + 16 * b + (lane & 15);
      int page = -1, slot = 0;
      if (at < v1) {
        slot = see.key(at);
        page = seq;
        if (a.table) {
          const int n = (int)args.page_size.quotient(slot);
          slot -= n * a.page_size;
          page = a.table[(int64_t)seq * a.table_width + n];
        }
      }
      const bool there = page >= 0 && page < a.pages;
      has[b] = ballot(there);
      const bool reads = there && inside;
      x.key[b] = *reinterpret_cast<const Words *>(
          reads ? key_codes + page * a.cache.key_page +
                      slot * a.cache.key_token : zeros);
      x.value[b] = *reinterpret_cast<const Words *>(
          reads ? value_codes + page * a.cache.value_page +
                      slot * a.cache.value_token : zeros);
      x.key_scale[b] = *(reads ? key_scales + page * args.scales.key_page +
                                     slot * args.scales.key_token : zeros);
      x.value_scale[b] = *(reads ? value_scales + page * args.scales.value_page +
                                       slot * args.scales.value_token : zeros);
    }
    x.none = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x.none |= (uint32_t)(~(has[i / 4] >> (4 * g + i % 4)) & 1) << i;
    return x;
  };

  v4f acc[kBlocks];
  float top, sum;
  float lower = 1.0f; // of this lane's row: a factor of the probabilities
  const uint32_t own = lds_address(lds) + wave * kWaveBytes;
  uint32_t across[2 * kBlocks];
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
      across[e * kBlocks + b] =
          own +
          Tile::place(16 * e + 4 * g + ((lane & 15) >> 2),
                      2 * b + ((lane & 3) >> 1)) + (lane & 1) * 8;

  bool some; // whether a key was there (wave-uniform)
  for (;;) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
      acc[b] = v4f{};
    top = -kInf;
    sum = 0.0f;
    some = false;
    for (int v = v0 + wave * kTile; v < v1; v += 4 * kTile) {
      const Data now = fetch(v);
      v4f score[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        score[b] = v4f{};
        const float by = fp4_scale(now.key_scale[b]);
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const v4u k = fp4_values(now.key[b][st], by);
#pragma unroll
          for (int i = kQueryParts<T> - 1; i >= 0; --i)
            score[b] = mma16(k, q[i][st], score[b]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((now.none >> i) & 1)
          score[i / 4][i % 4] = -kInf;
      float big = score[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i)
        big = fmaxf(big, score[i / 4][i % 4]);
      big = rows16_max(big) * scale;
      if (ballot(big > top) != 0) {
        const float to = fmaxf(top, big);
        const float by = to == -kInf ? 1.0f : __builtin_amdgcn_exp2f(top - to);
        top = to;
        sum *= by;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
          acc[b] *= by;
      }
      const float less = top == -kInf ? 0.0f : top;
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(score[i / 4][i % 4], scale, -less)) *
               lower;
        sum += p[i];
      }
      v4u weight[kWeightParts<T>];
      weight_parts(p, weight);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float by = fp4_scale(now.value_scale[b]);
#pragma unroll
        for (int w = 0; w < kWords; ++w)
          lds_write(own + Tile::place(16 * b + (lane & 15), kWords * g + w),
                    fp4_values(now.value[b][w], by));
      }
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const v2u x = lds_read_across(across[b], 0);
        const v2u y = lds_read_across(across[kBlocks + b], 0);
        const v4u vf = {x.x, x.y, y.x, y.y};
#pragma unroll
        for (int i = 0; i < kWeightParts<T>; ++i)
          acc[b] = mma16(vf, weight[i], acc[b]);
      }
      some |= ballot(((~now.none) & 0xFF) != 0) != 0;
    }
    // (a sum past fp32's range of values whose mean lies within: such rows once
    // more under lower probabilities, as in the attention of bf16 caches)
    const bool past = live && !all_finite(acc);
    if (ballot(past && lower == 1.0f) == 0)
      break;
    if (rows16_max(past ? 1.0f : 0.0f) != 0.0f)
      lower = __builtin_amdgcn_exp2f(-raise_of(v1 - v0));
  }
  const float raise = lower == 1.0f ? 0.0f : raise_of(v1 - v0);
  if (some && top == -kInf)
    top = kLowest;
  store_part<T, D, kWaveBytes>(a, lds, found, top, sum, raise, acc, rows, only,
                               seq, hk, first_row, a.sums + of * a.dim,
                               a.stats + of * 2);
}

// ---- host ------------------------------------------------------------------------

struct Plan {
  int64_t chunk, parts, rows, sums, stats; // sums, stats: floats
  int64_t bytes() const { return 4 * (sums + stats); }
};

Plan plan(int64_t sequences, int64_t capacity, int64_t query_heads,
          int64_t key_heads, int64_t d, int64_t window, int64_t sinks) {
  Plan p{};
  p.rows = sw::ceil_div(query_heads / key_heads, kRows) * kRows;
  const int64_t visible = most_visible(capacity, window, sinks);
  p.chunk = visible <= 512
                ? 512
                : part_of(visible, sequences * key_heads * (p.rows / kRows),
                          512, 256, 128);
  p.parts = std::max<int64_t>(1, sw::ceil_div(visible, p.chunk));
  if (p.parts > 1) {
    const int64_t all = sequences * key_heads * p.parts * p.rows;
    p.sums = all * (d <= 64 ? 64 : 128);
    p.stats = all * 2;
  }
  return p;
}

int check_all(int64_t sequences, int64_t pages, int64_t page_size,
              int64_t table_width, int64_t query_heads, int64_t key_heads,
              int64_t d, int64_t window, int64_t sinks, float alpha) {
  if (int rc = check_sizes(sequences, pages, page_size, table_width,
                           query_heads, key_heads, d, window, sinks, 0, alpha))
    return rc;
  return sw::check_fp4_heads(query_heads, key_heads, d);
}

template <typename T>
int fp4_step_entry(const int32_t *key_lengths, const int32_t *page_table,
                   const T *query, const uint8_t *key_codes,
                   const uint8_t *key_scales, const uint8_t *value_codes,
                   const uint8_t *value_scales, T *output, int64_t sequences,
                   int64_t pages, int64_t page_size, int64_t table_width,
                   int64_t query_heads, int64_t key_heads, int64_t d,
                   const int64_t *strides, int64_t window, int64_t sinks,
                   float alpha, void *workspace, int64_t workspace_bytes,
                   void *stream) {
  const char *what = "window attention decode fp4";
  sw::clear_error();
  if (!page_table)
    table_width = 1;
  if (int rc = check_all(sequences, pages, page_size, table_width, query_heads,
                         key_heads, d, window, sinks, alpha))
    return rc;
  if (int rc = sw::check_cache_sizes(sequences, 0, pages, page_size,
                                     table_width, page_table != nullptr))
    return rc;
  if (sequences > 0 && !key_lengths)
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "key lengths pointer is null");
  if (int rc = sw::check_value_alignment(4, {key_lengths, page_table}))
    return rc;
  int64_t packed[16];
  sw::fp4_packed_strides(packed, query_heads, key_heads, page_size, d);
  const int64_t *s = strides ? strides : packed;
  if (int rc = check_operand("query", query, {s[0], s[1]}, d, sizeof(T), false,
                             sequences, query_heads))
    return rc;
  if (int rc = check_operand("output", output, {s[2], s[3]}, d, sizeof(T), true,
                             sequences, query_heads))
    return rc;
  if (int rc = sw::check_fp4_cache("key", key_codes, key_scales, s + 4, d,
                                   pages, page_size, key_heads, false))
    return rc;
  if (int rc = sw::check_fp4_cache("value", value_codes, value_scales, s + 10,
                                   d, pages, page_size, key_heads, false))
    return rc;
  if (sequences == 0)
    return SW_OK;
  const Plan p = plan(sequences, page_size * table_width, query_heads,
                      key_heads, d, window, sinks);
  if (p.bytes() > 0 && (!workspace || !sw::aligned16(workspace) ||
                        workspace_bytes < p.bytes()))
    return sw::fail(SW_ERR_INVALID_ARGUMENT,
                    "%s needs a 16-byte aligned workspace of %lld bytes", what,
                    (long long)p.bytes());
  Fp4StepArgs args{};
  StepArgs &a = args.s;
  a.lengths = key_lengths;
  a.table = page_table;
  a.query = query;
  a.output = output;
  a.cache = {key_codes, value_codes, s[4], s[5], s[6], s[10], s[11], s[12]};
  args.scales = {key_scales, value_scales, s[7], s[8], s[9],
                 s[13], s[14], s[15]};
  args.page_size = Divisor((uint32_t)page_size);
  a.query_token = s[0];
  a.query_head = s[1];
  a.output_token = s[2];
  a.output_head = s[3];
  a.sequences = (int)sequences;
  a.pages = (int)pages;
  a.page_size = (int)page_size;
  a.table_width = (int)table_width;
  a.query_heads = (int)query_heads;
  a.key_heads = (int)key_heads;
  a.group = (int)(query_heads / key_heads);
  a.d = (int)d;
  a.dim = d <= 64 ? 64 : 128;
  a.window = (int)std::min<int64_t>(window, sw::kMostTokens);
  a.sinks = (int)std::min<int64_t>(sinks, sw::kMostTokens);
  a.alpha = alpha;
  a.chunk = (int)p.chunk;
  a.parts = (int)p.parts;
  a.rows = (int)p.rows;
  a.lower = std::ldexp(
      1.0f, -(int)std::ceil(std::log2((double)(p.chunk * p.parts))) - 1);
  a.sums = static_cast<float *>(workspace);
  a.stats = a.sums + p.sums;
  const int64_t grid = sequences * key_heads * (p.rows / kRows) * p.parts;
  const int64_t join = sequences * query_heads;
  if (int rc = sw::check_flat_grid(std::max(grid, join), kThreads, what))
    return rc;
  const hipStream_t st = sw::as_stream(stream);
  const dim3 g((unsigned)grid);
  if (d <= 64)
    fp4_cache_parts<T, 64><<<g, kThreads, 0, st>>>(args);
  else
    fp4_cache_parts<T, 128><<<g, kThreads, 0, st>>>(args);
  if (int rc = sw::launch_check(what))
    return rc;
  if (p.parts == 1)
    return SW_OK;
  if (d <= 64)
    window_cache_join<T, 64><<<dim3((unsigned)join), kThreads, 0, st>>>(a);
  else
    window_cache_join<T, 128><<<dim3((unsigned)join), kThreads, 0, st>>>(a);
  return sw::launch_check(what);
}

} // namespace

extern "C" int64_t sw_window_attention_decode_fp4_workspace_bytes(
    int64_t sequences, int64_t page_size, int64_t table_width,
    int64_t query_heads, int64_t key_heads, int64_t d, int64_t window,
    int64_t sinks) {
  if (sequences == 0 ||
      check_all(sequences, 0, page_size, table_width, query_heads, key_heads, d,
                window, sinks, 0.0f) != SW_OK)
    return 0;
  return plan(sequences, page_size * table_width, query_heads, key_heads, d,
              window, sinks).bytes();
}

extern "C" int sw_window_attention_decode_fp4_f32(
    const int32_t *key_lengths, const int32_t *page_table, const float *query,
    const uint8_t *key_codes, const uint8_t *key_scales,
    const uint8_t *value_codes, const uint8_t *value_scales, float *output,
    int64_t sequences, int64_t pages, int64_t page_size, int64_t table_width,
    int64_t query_heads, int64_t key_heads, int64_t d, const int64_t *strides,
    int64_t window, int64_t sinks, float alpha, void *workspace,
    int64_t workspace_bytes, void *stream) {
  return fp4_step_entry<float>(
      key_lengths, page_table, query, key_codes, key_scales, value_codes,
      value_scales, output, sequences, pages, page_size, table_width,
      query_heads, key_heads, d, strides, window, sinks, alpha, workspace,
      workspace_bytes, stream);
}

extern "C" int sw_window_attention_decode_fp4_bf16(
    const int32_t *key_lengths, const int32_t *page_table,
    const uint16_t *query, const uint8_t *key_codes, const uint8_t *key_scales,
    const uint8_t *value_codes, const uint8_t *value_scales, uint16_t *output,
    int64_t sequences, int64_t pages, int64_t page_size, int64_t table_width,
    int64_t query_heads, int64_t key_heads, int64_t d, const int64_t *strides,
    int64_t window, int64_t sinks, float alpha, void *workspace,
    int64_t workspace_bytes, void *stream) {
  return fp4_step_entry<uint16_t>(
      key_lengths, page_table, query, key_codes, key_scales, value_codes,
      value_scales, output, sequences, pages, page_size, table_width,
      query_heads, key_heads, d, strides, window, sinks, alpha, workspace,
      workspace_bytes, stream);
}
