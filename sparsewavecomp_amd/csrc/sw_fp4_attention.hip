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
//
// Tiles start at multiples of 32 keys, so that a half of 16 lies in one page
// wherever a page holds a multiple of 16: its addresses are then scalar ones
// plus a lane's constant offset.  Halves that cross a page's end take each
// lane's own.  The pages of a wave's next 32 tiles are found at once, a half by
// each lane; the next tile is on its way while one is multiplied.
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
  const int t0 = part * (a.chunk / kTile);
  const int t1 = see.tiles() < t0 + a.chunk / kTile ? see.tiles()
                                                    : t0 + a.chunk / kTile;
  const int64_t of =
      (((int64_t)seq * a.key_heads + hk) * a.parts + part) * a.rows + first_row;
  const bool only = a.parts == 1;
  if (t1 <= t0 && !only)
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

  // This lane's quarter of a row: codes, and the scale of its block.  Quarters
  // past d read the row's first one; the queries are zero there, and so is the
  // scale.
  const bool inside = D / 4 * g < a.d;
  const int code_at = inside ? D / 8 * g : 0, scale_at = inside ? D * g / 128 : 0;
  const int row_of = lane & 15;
  const Scales &sc = args.scales;
  const uint8_t *key_codes =
      static_cast<const uint8_t *>(a.cache.key) + hk * a.cache.key_head;
  const uint8_t *value_codes =
      static_cast<const uint8_t *>(a.cache.value) + hk * a.cache.value_head;
  const uint8_t *key_scales = sc.key + hk * sc.key_head;
  const uint8_t *value_scales = sc.value + hk * sc.value_head;
  // (a token stride is at most 2^23)
  const uint32_t key_off = row_of * (uint32_t)a.cache.key_token + code_at;
  const uint32_t value_off = row_of * (uint32_t)a.cache.value_token + code_at;
  const uint32_t key_scale_off = row_of * (uint32_t)sc.key_token + scale_at;
  const uint32_t value_scale_off = row_of * (uint32_t)sc.value_token + scale_at;

  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  struct Data {
    Words key[2], value[2];
    uint32_t key_scale[2], value_scale[2];
    uint32_t has; // bit i: key i of the tile is seen (wave-uniform)
  };
  struct Halves { // of the wave's next tiles: lane l has half l % 2 of l / 2
    int page, slot; // of its first key; page -1: it is not there
  };
  auto page_of = [&](int key, int &slot) __attribute__((always_inline)) {
    int page = seq;
    slot = key;
    if (a.table) {
      const int n = (int)args.page_size.quotient(key);
      slot -= n * a.page_size;
      page = a.table[(int64_t)seq * a.table_width + n];
    }
    return page >= 0 && page < a.pages ? page : -1;
  };
  auto locate = [&](int first) __attribute__((always_inline)) {
    const int tile = first + 4 * (lane >> 1);
    const int key = see.tile_key(tile) + 16 * (lane & 1);
    Halves h{-1, 0};
    if (tile < t1 && key < see.end())
      h.page = page_of(key, h.slot);
    return h;
  };
  auto load = [&](Data &x, int b, int64_t kc, int64_t vc, int64_t ks,
                  int64_t vs) __attribute__((always_inline)) {
    x.key[b] = *reinterpret_cast<const Words *>(key_codes + kc);
    x.value[b] = *reinterpret_cast<const Words *>(value_codes + vc);
    x.key_scale[b] = key_scales[ks];
    x.value_scale[b] = value_scales[vs];
  };
  // tile k of `h`, whose first key is `key`
  auto fetch = [&](const Halves &h, int k, int key)
                   __attribute__((always_inline)) {
    Data x;
    x.has = 0;
#pragma unroll
    for (int b = 0; b < 2; ++b, key += 16) {
      const int64_t page = __builtin_amdgcn_readlane(h.page, 2 * k + b);
      const int64_t slot = __builtin_amdgcn_readlane(h.slot, 2 * k + b);
      x.key[b] = x.value[b] = Words{};
      x.key_scale[b] = x.value_scale[b] = 0;
      if (slot + 16 <= a.page_size) {
        if (page < 0)
          continue;
        const uint8_t *kc = key_codes + (page * a.cache.key_page +
                                         slot * a.cache.key_token);
        const uint8_t *vc = value_codes + (page * a.cache.value_page +
                                           slot * a.cache.value_token);
        const uint8_t *ks =
            key_scales + (page * sc.key_page + slot * sc.key_token);
        const uint8_t *vs =
            value_scales + (page * sc.value_page + slot * sc.value_token);
        x.key[b] = *reinterpret_cast<const Words *>(kc + key_off);
        x.value[b] = *reinterpret_cast<const Words *>(vc + value_off);
        x.key_scale[b] = ks[key_scale_off];
        x.value_scale[b] = vs[value_scale_off];
        const bool all = (key + 16 <= see.lead || key >= see.start) &&
                         key + 16 <= see.end();
        x.has |= (all ? 0xFFFFu
                      : (uint32_t)ballot(see.sees(key + row_of)) & 0xFFFFu)
                 << (16 * b);
      } else {
        int s = 0, p = -1;
        if (see.sees(key + row_of))
          p = page_of(key + row_of, s);
        if (p >= 0)
          load(x, b, p * a.cache.key_page + s * a.cache.key_token + code_at,
               p * a.cache.value_page + s * a.cache.value_token + code_at,
               p * sc.key_page + s * sc.key_token + scale_at,
               p * sc.value_page + s * sc.value_token + scale_at);
        x.has |= ((uint32_t)ballot(p >= 0) & 0xFFFFu) << (16 * b);
      }
    }
    return x;
  };

  v4f acc[kBlocks], total; // total: the probabilities' sums, in all four
  float top;
  float lower = 1.0f; // of this lane's row: a factor of the probabilities
  bool again = false; // whether a row has such a factor (wave-uniform)
  const uint32_t own = lds_address(lds) + wave * kWaveBytes;
  // of a read across rows 4 g + .. and of a write: chunks differ by what the
  // swizzle leaves alone, rows 16 apart have the same
  uint32_t across = own +
                    Tile::place(4 * g + (row_of >> 2), (lane & 3) >> 1) +
                    (lane & 1) * 8;
  uint32_t along = own + Tile::place(row_of, kWords * g);
  const v4u ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

  auto compute = [&](Data &x) __attribute__((always_inline)) {
    // (keeps the compiler from holding every address in a register)
    asm volatile("" : "+v"(across), "+v"(along));
    v4f score[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      score[b] = v4f{};
      const float by = fp4_scale(inside ? x.key_scale[b] : 0u);
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const v4u k = fp4_values(x.key[b][st], by);
#pragma unroll
        for (int i = kQueryParts<T> - 1; i >= 0; --i)
          score[b] = mma16(k, q[i][st], score[b]);
      }
    }
    if (x.has != 0xFFFFFFFFu) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!((x.has >> (16 * (i / 4) + 4 * g + i % 4)) & 1))
          score[i / 4][i % 4] = -kInf;
      // (what lies at a place that is not seen may be NaN)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        if (!((x.has >> (16 * b + row_of)) & 1))
          x.value_scale[b] = 0;
    }
    float big = score[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i)
      big = fmaxf(big, score[i / 4][i % 4]);
    big = rows16_max(big) * scale;
    if (ballot(big > top) != 0) {
      const float to = fmaxf(top, big);
      const float by = to == -kInf ? 1.0f : __builtin_amdgcn_exp2f(top - to);
      top = to;
      total *= by;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        acc[b] *= by;
    }
    const float less = top == -kInf ? 0.0f : top;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      p[i] = __builtin_amdgcn_exp2f(fmaf(score[i / 4][i % 4], scale, -less));
    if (again) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        p[i] *= lower;
    }
    v4u weight[kWeightParts<T>];
    weight_parts(p, weight);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float by = fp4_scale(x.value_scale[b]);
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        lds_write((along ^ (w << 4)) + 16 * b * Tile::kPitch,
                  fp4_values(x.value[b][w], by));
    }
#pragma unroll
    for (int i = 0; i < kWeightParts<T>; ++i)
      total = mma16(ones, weight[i], total);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const v2u lo = lds_read_across(across ^ (b << 5), 0);
      const v2u hi = lds_read_across(across ^ (b << 5), 16 * Tile::kPitch);
      const v4u vf = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int i = 0; i < kWeightParts<T>; ++i)
        acc[b] = mma16(vf, weight[i], acc[b]);
    }
  };

  bool some; // whether a key was there (wave-uniform)
  const int mine = t1 - t0 > wave ? (t1 - t0 - wave + 3) / 4 : 0;
  for (;;) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
      acc[b] = v4f{};
    total = v4f{};
    top = -kInf;
    some = false;
    for (int done = 0; done < mine; done += kWave / 2) {
      const int first = t0 + wave + 4 * done;
      const int n = mine - done < kWave / 2 ? mine - done : kWave / 2;
      const Halves h = locate(first);
      Data x = fetch(h, 0, see.tile_key(first)), y;
      for (int k = 0; k < n; k += 2) {
        if (k + 1 < n)
          y = fetch(h, k + 1, see.tile_key(first + 4 * k + 4));
        some |= x.has != 0;
        compute(x);
        if (k + 1 < n) {
          if (k + 2 < n)
            x = fetch(h, k + 2, see.tile_key(first + 4 * k + 8));
          some |= y.has != 0;
          compute(y);
        }
      }
    }
    // (a sum past fp32's range of values whose mean lies within: such rows once
    // more under lower probabilities, as in the attention of bf16 caches)
    const bool past = live && !all_finite(acc);
    if (again || ballot(past) == 0)
      break;
    again = true;
    if (rows16_max(past ? 1.0f : 0.0f) != 0.0f)
      lower = __builtin_amdgcn_exp2f(-raise_of((t1 - t0) * kTile));
  }
  const float raise = lower == 1.0f ? 0.0f : raise_of((t1 - t0) * kTile);
  if (some && top == -kInf)
    top = kLowest;
  store_part<T, D, kWaveBytes>(a, lds, found, top, total[0], raise, acc, rows,
                               only, seq, hk, first_row, a.sums + of * a.dim,
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
  // Tiles of 32 keys hold less than they might at both ends of the window and
  // behind the sinks.
  const int64_t tiled =
      std::min(visible + 3 * (kTile - 1), sw::ceil_div(capacity, kTile) * kTile);
  p.chunk = visible <= 512
                ? 640
                : part_of(tiled, sequences * key_heads * (p.rows / kRows),
                          512, 256, 128);
  p.parts = std::max<int64_t>(1, sw::ceil_div(tiled, p.chunk));
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
  a.by_tiles = true;
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
