// Attention of one query for each sequence against a key-value cache, over a
// sliding window with sinks or behind a prefix that all sequences share, on
// gfx950.
//
// Every visible key and value is read once for the query heads that share its
// head: with G of them a key of d elements takes part in 4 G d operations for
// 2 d elements read, so memory bounds these kernels.  A sequence's keys are cut
// into chunks, one workgroup each, and the chunks' (m, l, o) joined:
//   m = max m_c,  w_c = l_c 2^(m_c - m),  l = sum w_c,  o = sum o_c w_c / l,
// o_c being a chunk's weighted mean: sums of values, which fp32 may not hold
// where their mean is finite, stay within a chunk, which sees whether they did.
// The prefix is cut the same way; its rows are the query heads of all
// sequences together.
#include "sw_heads.h"
#include "sw_internal.h"

#include <algorithm>
#include <cmath>

using namespace swd;
using sw::Operand;
using sw::check_operand;

namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kInf = __builtin_inff();
// the maximum of keys whose scores are all -inf: the result is NaN then, where
// it is zero without a key (a maximum of -inf)
constexpr float kLowest = -3.402823466e+38f;
constexpr int kThreads = 256; // four waves
constexpr int kRows = 16;     // query rows of a workgroup's part
constexpr int kTile = 32;     // keys a wave takes at a time

// what lanes without a key read
__device__ const uint32_t kZeros[8] = {};

struct Cache {
  const void *key, *value;
  int64_t key_page, key_token, key_head; // strides in elements
  int64_t value_page, value_token, value_head;
};

struct StepArgs {
  const int32_t *lengths, *table; // table may be null: page i is sequence i's
  const void *query;
  void *output;
  Cache cache, prefix; // (the prefix: one page)
  int64_t query_token, query_head, output_token, output_head;
  int sequences, pages, page_size, table_width;
  int query_heads, key_heads, group, d, dim; // dim: d padded to 64 or 128
  int window, sinks, prefix_tokens;
  float alpha;
  // Parts of `chunk` keys: `parts` at most for a sequence, `prefix_parts` of
  // the prefix, whose query rows are those of all sequences.  A part of rows
  // leaves o in [part][rows][dim] and (m, l) in [part][rows][2].
  int chunk, parts, prefix_chunk, prefix_parts;
  int rows, prefix_rows; // of one part: a multiple of 16, of 16 or 128
  // a power of two: the number of all keys times it is below 1
  float lower;
  float *sums, *stats, *prefix_sums, *prefix_stats;
  // workgroups of the prefix: by cache_part and by prefix_part
  int64_t prefix_items, wide_items;
};

// The keys that sequence i's query sees: the first `lead`, and those from
// `start` on, `count` in all.
struct Visible {
  int lead, start, count;
  __device__ __forceinline__ Visible(const StepArgs &a, int i) {
    const int64_t room = (int64_t)a.page_size * a.table_width;
    int n = a.lengths[i];
    n = n < 0 ? 0 : n > room ? (int)room : n;
    start = n > a.window ? n - a.window : 0;
    lead = a.sinks < start ? a.sinks : start;
    count = lead + n - start;
  }
  __device__ __forceinline__ int key(int v) const {
    return v < lead ? v : v - lead + start;
  }
};

__device__ __forceinline__ float rows16_max(float v) { // over lanes l % 16
  return both_halves_max(fmaxf(v, swizzle_xor16(v)));
}
__device__ __forceinline__ float rows16_sum(float v) {
  return both_halves_sum(v + swizzle_xor16(v));
}
__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(lane * 4, (int)v);
  const int hi = __builtin_amdgcn_ds_bpermute(lane * 4, (int)(v >> 32));
  return (int64_t)hi << 32 | lo;
}

// One chunk of keys against up to 16 query rows: 16 x 16 products of K Q^T, 32
// keys a wave at a time; V goes through LDS to be read across its rows.  The
// four waves' results are joined in LDS.  The keys of a wave's next tile are
// not fetched ahead: the registers hold another wave a SIMD instead, whose
// fetches go on meanwhile (64 sequences, window 4096: 201 us with two waves
// and fetches ahead, 195 us with three; four waves' registers spill, 306 us).
// Memory bounds it: those 64 read 5.5 TB/s, 4 sequences of 65,536 keys take
// 170 us, 5.3 TB/s (a kernel that only reads: 6.5); one of 260 keys 6.8 us, a
// chain of trips.
template <typename T, int D> struct CacheParts {
  using Tile = RowTile<T, D, kTile, kWave>;
  static constexpr int kWaveBytes =
      Tile::kBytes > kRows * D * 4 ? Tile::kBytes : kRows * D * 4;
  static constexpr int kBytes = 4 * kWaveBytes;
  // (bf16 rows of up to 64, 64 sequences, window 4096: 114 us with four waves,
  // 104 with five)
  static constexpr int kWaves =
      sizeof(T) * D > 256 ? 1 : sizeof(T) * D > 128 ? 3 : 5;
};
struct Totals {
  float top[4][kRows], sum[4][kRows], raise[4][kRows];
};

template <typename T, int D, bool SPLIT>
__device__ __forceinline__ void cache_part(const StepArgs &a, int64_t item,
                                           char *lds, Totals &found) {
  using Tile = RowTile<T, D, kTile, kWave>;
  constexpr int kSteps = D / 32;  // products along d
  constexpr int kBlocks = D / 16; // output rows of 16
  constexpr int kPieces = Tile::kBytes / 1024;
  constexpr int kPieceRows = 1024 / Tile::kPitch;
  constexpr int kWaveBytes = CacheParts<T, D>::kWaveBytes;

  const int lane = lane_id(), g = lane >> 4, wave = wave_in_group();
  // ---- which rows, which keys
  const bool shared = item < a.prefix_items;
  int hk, part, first_row, rows, total, v0, v1, seq = 0;
  float *sums, *stats;
  Visible see(a, 0);
  if (shared) {
    part = (int)(item % a.prefix_parts);
    item /= a.prefix_parts;
    first_row = (int)(item % (a.prefix_rows / kRows)) * kRows;
    hk = (int)(item / (a.prefix_rows / kRows));
    total = a.sequences * a.group;
    v0 = part * a.prefix_chunk;
    v1 = a.prefix_tokens < v0 + a.prefix_chunk ? a.prefix_tokens
                                               : v0 + a.prefix_chunk;
    const int64_t of =
        ((int64_t)hk * a.prefix_parts + part) * a.prefix_rows + first_row;
    sums = a.prefix_sums + of * a.dim;
    stats = a.prefix_stats + of * 2;
  } else {
    item -= a.prefix_items;
    part = (int)(item % a.parts);
    item /= a.parts;
    first_row = (int)(item % (a.rows / kRows)) * kRows;
    item /= a.rows / kRows;
    hk = (int)(item % a.key_heads);
    seq = (int)(item / a.key_heads);
    see = Visible(a, seq);
    total = a.group;
    v0 = part * a.chunk;
    v1 = see.count < v0 + a.chunk ? see.count : v0 + a.chunk;
    const int64_t of =
        (((int64_t)seq * a.key_heads + hk) * a.parts + part) * a.rows +
        first_row;
    sums = a.sums + of * a.dim;
    stats = a.stats + of * 2;
  }
  const bool only = a.parts == 1 && a.prefix_parts == 0;
  if (v1 <= v0 && !only)
    return;
  rows = total - first_row < kRows ? total - first_row : kRows;

  const bool none = a.alpha == 0.0f;
  const float scale = none ? 1.0f : fabsf(a.alpha) * kLog2e;
  Frag<T> q[kSteps];
  const int my_row = first_row + (lane & 15); // query row of this lane
  const bool live = (lane & 15) < rows;
  {
    const int row = live ? my_row : first_row;
    const int i = shared ? row / a.group : seq;
    const int head = hk * a.group + (shared ? row % a.group : row);
    const T *p = static_cast<const T *>(a.query) + i * a.query_token +
                 head * a.query_head;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int c = 32 * st + 8 * g;
      q[st] = live && c < a.d && !none ? ld_frag(p + c) : zero_frag<T>();
      if (a.alpha < 0.0f)
        q[st] = negate_frag<T>(q[st]);
    }
  }

  const Cache &from = shared ? a.prefix : a.cache;
  const T *keys = static_cast<const T *>(from.key) + hk * from.key_head;
  const T *values = static_cast<const T *>(from.value) + hk * from.value_head;
  const T *zeros = reinterpret_cast<const T *>(kZeros);
  struct Rows { int64_t key, value; }; // -1: no key
  // the rows of this lane's key (l % 32) of the tile from v on
  auto rows_of = [&](int v) __attribute__((always_inline)) {
    v += lane & 31;
    Rows r{-1, -1};
    if (v < v1) {
      int64_t page = 0;
      uint32_t slot = v;
      if (!shared) {
        slot = see.key(v);
        page = seq;
        if (a.table) {
          const uint32_t n = slot / (uint32_t)a.page_size;
          slot -= n * a.page_size;
          page = a.table[(int64_t)seq * a.table_width + n];
        }
      }
      if (shared || (page >= 0 && page < a.pages))
        r = {page * from.key_page + slot * from.key_token,
             page * from.value_page + slot * from.value_token};
    }
    return r;
  };
  struct Data {
    Frag<T> k[2][kSteps];
    v4u v[kPieces];
    uint32_t none; // bit i: this lane's key i of the products is none
  };
  auto fetch = [&](const Rows &r) __attribute__((always_inline)) {
    Data x;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t row = lane_value(r.key, 16 * b + (lane & 15));
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const int c = 32 * st + 8 * g;
        x.k[b][st] = ld_frag(row >= 0 && c < a.d ? keys + row + c : zeros);
      }
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int64_t row =
          lane_value(r.value, p * kPieceRows + lane / Tile::kChunks);
      const int c = lane % Tile::kChunks * (16 / (int)sizeof(T));
      x.v[p] = *reinterpret_cast<const v4u *>(
          row >= 0 && c < a.d ? values + row + c : zeros);
    }
    const uint64_t has = ballot(r.key >= 0);
    x.none = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x.none |= (uint32_t)(~(has >> (16 * (i / 4) + 4 * g + i % 4)) & 1) << i;
    return x;
  };

  v4f acc[kBlocks];
  float top, sum;
  float lower = 1.0f; // of this lane's row: a factor of the probabilities
  const uint32_t own = lds_address(lds) + wave * kWaveBytes;
  uint32_t across[sizeof(T) == 2 ? 2 * kBlocks : 1]; // (bf16)
  if constexpr (sizeof(T) == 2) {
    const int i = lane & 15;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        across[e * kBlocks + b] =
            own + Tile::place(16 * e + 4 * g + (i >> 2), 2 * b + ((i & 3) >> 1)) +
            (i & 1) * 8;
  }

  bool some; // whether a key was there (wave-uniform)
  for (;;) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
      acc[b] = v4f{};
    top = -kInf;
    sum = 0.0f;
    some = false;
    int v = v0 + wave * kTile;
    while (v < v1) {
      const Data now = fetch(rows_of(v));
      v4f score[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        score[b] = v4f{};
#pragma unroll
        for (int st = 0; st < kSteps; ++st)
          score[b] = mma16(now.k[b][st], q[st], score[b]);
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
      // bf16: the matrix core takes the probabilities as two bf16 parts, 15 bits
      // of them together, for which it has the time (3.6 % busy with one part;
      // 64 sequences, window 4096: 194.5 us, 192.2 with one; 4 of 65,536 keys:
      // 179.4, 180.5).  Beside a prefix's products it has not (SPLIT, 128
      // sequences behind 16,384 keys: 182.8 us, 177.0 with one): they round to
      // bf16 there, as the prefix's do.  Their sum does not.
      Frag<T> pf, rest;
      if constexpr (SPLIT)
        split_frag(p, pf, rest);
      else
        pf = make_frag<T>(p);
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        lds_write(own + Tile::place(i * kPieceRows + lane / Tile::kChunks,
                                    lane % Tile::kChunks), now.v[i]);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        Frag<T> vf;
        if constexpr (sizeof(T) == 2) {
          const v2u x = lds_read_across(across[b], 0);
          const v2u y = lds_read_across(across[kBlocks + b], 0);
          vf = v4u{x.x, x.y, y.x, y.y};
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int c = 16 * b + (lane & 15);
            vf[i] = lds_read<float>(
                own + Tile::place(16 * (i >> 2) + 4 * g + (i & 3), c >> 2) +
                (c & 3) * 4, 0);
          }
        }
        acc[b] = mma16(vf, pf, acc[b]);
        if constexpr (SPLIT)
          acc[b] = mma16(vf, rest, acc[b]);
      }
      some |= ballot(((~now.none) & 0xFF) != 0) != 0;
      v += 4 * kTile;
    }
    // A sum past fp32's range of values whose mean lies within: such rows once
    // more, under probabilities that are lower by the number of keys.  (Of them
    // alone, what is below that factor times 2^-126 of the largest probability,
    // or such a value, is lost.)
    const bool past = live && !all_finite(acc);
    if (ballot(past && lower == 1.0f) == 0)
      break;
    if (rows16_max(past ? 1.0f : 0.0f) != 0.0f)
      lower = __builtin_amdgcn_exp2f(-raise_of(v1 - v0));
  }
  const float raise = lower == 1.0f ? 0.0f : raise_of(v1 - v0);
  if (some && top == -kInf)
    top = kLowest;

  // ---- the four waves' results, joined
  sum = rows16_sum(sum);
  if (g == 0) {
    found.top[wave][lane] = top;
    found.sum[wave][lane] = sum;
    found.raise[wave][lane] = raise;
  }
  // o[row][d] of each wave, in its own part of LDS
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
    lds_write(own + ((lane & 15) * D + 16 * b + 4 * g) * 4, acc[b]);
  __syncthreads();
  for (int x = threadIdx.x; x < kRows * D / 4; x += kThreads) {
    const int r = x / (D / 4), c = x % (D / 4) * 4;
    if (r >= rows)
      break;
    float m = found.top[0][r], most = found.raise[0][r];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      m = fmaxf(m, found.top[w][r]);
      most = fmaxf(most, found.raise[w][r]);
    }
    most += 3.0f; // (four sums that are finite have a finite sum)
    float l = 0.0f;
    v4f o = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float by =
          found.top[w][r] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(found.top[w][r] - m);
      by *= __builtin_amdgcn_exp2f(found.raise[w][r] - most);
      const v4f y =
          lds_read<v4f>(lds_address(lds) + w * kWaveBytes + (r * D + c) * 4, 0);
      l = fmaf(found.sum[w][r], by, l);
      o += y * by;
    }
    if (only) {
      if (c < a.d) {
        const bool empty = m == -kInf;
        const float by = 1.0f / l;
        T *out = static_cast<T *>(a.output) + seq * a.output_token +
                 (hk * a.group + first_row + r) * a.output_head + c;
        st4(out, empty ? 0.0f : o[0] * by, empty ? 0.0f : o[1] * by,
            empty ? 0.0f : o[2] * by, empty ? 0.0f : o[3] * by);
      }
    } else {
      if (l != 0.0f) // (zero: no key, or scores of -inf alone)
        o *= 1.0f / l;
      *reinterpret_cast<v4f *>(sums + r * D + c) = o;
      if (c == 0) {
        stats[2 * r] = m;
        stats[2 * r + 1] = l * __builtin_amdgcn_exp2f(most);
      }
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, (CacheParts<T, D>::kWaves)) void
window_cache_parts(StepArgs a) {
  __shared__ __align__(1024) char lds[CacheParts<T, D>::kBytes];
  __shared__ Totals found;
  cache_part<T, D, sizeof(T) == 2>(a, blockIdx.x, lds, found);
}

// The prefix against many query rows: 128 rows, 32 a wave, and one chunk of
// the prefix, in tiles of LDS that the four waves share; 32 x 32 products of
// K Q^T as in the window's forward pass.
template <typename T, int D> struct Prefix {
  static constexpr int kTile = sizeof(T) == 2 ? 64 : 32;
  using Tile = RowTile<T, D, kTile, kThreads>;
  static constexpr int kSteps = D / 16;
  static constexpr int kBlocks = D / 32;
  static constexpr int kKeyBlocks = kTile / 32;
  // (fp32 rows of up to 64, 64 sequences behind 4,096 keys: 65 us with two
  // waves, 47 with three)
  static constexpr int kWaves =
      sizeof(T) * D > 256 ? 1 : sizeof(T) == 4 ? 3 : 2;
  static constexpr int kBytes = std::max(4 * Tile::kBytes,
                                         CacheParts<T, D>::kBytes);
};
constexpr int kPrefixRows = 128;

template <typename T, int D>
__device__ __forceinline__ void prefix_part(const StepArgs &a, int64_t item,
                                            char *lds, int *verdict) {
  using F = Prefix<T, D>;
  using Tile = typename F::Tile;
  constexpr int KT = F::kTile;

  const int tiles = a.prefix_rows / kPrefixRows;
  const int first_row = (int)(item % tiles) * kPrefixRows;
  item /= tiles;
  const int part = (int)(item % a.prefix_parts);
  const int hk = (int)(item / a.prefix_parts);
  const int v0 = part * a.prefix_chunk;
  const int v1 = a.prefix_tokens < v0 + a.prefix_chunk ? a.prefix_tokens
                                                       : v0 + a.prefix_chunk;
  const int count = (v1 - v0 + KT - 1) / KT;

  const int lane = lane_id(), h = lane >> 5, wave = wave_in_group();
  const int row = first_row + 32 * wave + (lane & 31);
  const bool live = row < a.sequences * a.group;
  const bool none = a.alpha == 0.0f;
  const float scale = none ? 1.0f : fabsf(a.alpha) * kLog2e;
  Frag<T> q[F::kSteps];
  {
    const int r = live ? row : 0;
    const T *p = static_cast<const T *>(a.query) +
                 r / a.group * a.query_token +
                 (hk * a.group + r % a.group) * a.query_head;
    load_rows<T>(q, p, live && !none, a.d, a.alpha < 0.0f);
  }
  const T *keys = static_cast<const T *>(a.prefix.key) + hk * a.prefix.key_head;
  const T *values =
      static_cast<const T *>(a.prefix.value) + hk * a.prefix.value_head;
  const uint32_t kbytes = (uint32_t)(a.prefix.key_token * sizeof(T));
  const uint32_t vbytes = (uint32_t)(a.prefix.value_token * sizeof(T));
  const typename Tile::Lane at;
  const uint32_t base = lds_address(lds);
  auto copy = [&](int t) __attribute__((always_inline)) {
    const int64_t j = v0 + t * KT;
    const uint32_t to = base + (t & 1) * 2 * Tile::kBytes;
    Tile::copy(to, keys + j * a.prefix.key_token, v1 - (int)j, kbytes, a.d, wave);
    Tile::copy(to + Tile::kBytes, values + j * a.prefix.value_token,
               v1 - (int)j, vbytes, a.d, wave);
  };

  v16f acc[F::kBlocks];
  float top, sum;
  float raise = 0.0f; // as in cache_part
  // (waves without rows only copy)
  const bool work = first_row + 32 * wave < a.sequences * a.group;
  auto step = [&](int t, auto parity, auto careful)
                  __attribute__((always_inline)) {
    landed();
    if (t + 1 < count)
      copy(t + 1);
    if (!work)
      return;
    const uint32_t kt = base + decltype(parity)::value * 2 * Tile::kBytes;
    const uint32_t vt = kt + Tile::kBytes;
    v16f score[F::kKeyBlocks];
#pragma unroll
    for (int kb = 0; kb < F::kKeyBlocks; ++kb) {
      score[kb] = v16f{};
#pragma unroll
      for (int st = 0; st < F::kSteps; ++st)
        score[kb] = mma32(Tile::along(kt, at, kb, st), q[st], score[kb]);
    }
    const int left = v1 - (v0 + t * KT) - 4 * h;
    if (left < KT) {
#pragma unroll
      for (int kb = 0; kb < F::kKeyBlocks; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          score[kb][r] = 32 * kb + 8 * (r >> 2) + (r & 3) < left
                             ? score[kb][r] : -kInf;
    }
    float big = score[0][0];
#pragma unroll
    for (int kb = 0; kb < F::kKeyBlocks; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        big = fmaxf(big, score[kb][r]);
    big = both_halves_max(big) * scale;
    if (ballot(big > top + 8.0f) != 0) { // (as in the window's forward pass)
      const float to = fmaxf(top, big);
      const float by = to == -kInf ? 1.0f : __builtin_amdgcn_exp2f(top - to);
      top = to;
      sum *= by;
#pragma unroll
      for (int b = 0; b < F::kBlocks; ++b)
        acc[b] *= by;
    }
    const float less = top == -kInf ? 0.0f : top;
    const float lower = __builtin_amdgcn_exp2f(-raise);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kb = 0; kb < F::kKeyBlocks; ++kb) {
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
        const Frag<T> pf = make_frag<T>(p + 8 * half);
#pragma unroll
        for (int b = 0; b < F::kBlocks; ++b)
          acc[b] = mma32(Tile::across(vt, at, 2 * kb + half, b), pf, acc[b]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto pass = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < F::kBlocks; ++b)
      acc[b] = v16f{};
    top = -kInf;
    sum = 0.0f;
    if (count > 0)
      copy(0);
    for (int t = 0; t < count; t += 2) {
      step(t, std::integral_constant<int, 0>{}, careful);
      if (t + 1 < count)
        step(t + 1, std::integral_constant<int, 1>{}, careful);
    }
  };
  pass(std::false_type{});
  // (as in cache_part; the maximum lags by up to 2^8 here)
  const bool past = live && !all_finite(acc);
  if (any_wave(past, verdict)) {
    if (both_halves_max(past ? 1.0f : 0.0f) != 0.0f)
      raise = 8.0f + raise_of(v1 - v0);
    pass(std::true_type{});
  }
  sum = both_halves_sum(sum);
  if (!live)
    return;
  if (top == -kInf)
    top = kLowest;
  if (sum != 0.0f) {
    const float by = 1.0f / sum;
#pragma unroll
    for (int b = 0; b < F::kBlocks; ++b)
      acc[b] *= by;
  }
  const int64_t of = ((int64_t)hk * a.prefix_parts + part) * a.prefix_rows + row;
#pragma unroll
  for (int b = 0; b < F::kBlocks; ++b)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      st4(a.prefix_sums + of * D + 32 * b + 8 * (r >> 2) + 4 * h, acc[b][r],
          acc[b][r + 1], acc[b][r + 2], acc[b][r + 3]);
  if (h == 0) {
    a.prefix_stats[2 * of] = top;
    a.prefix_stats[2 * of + 1] = sum * __builtin_amdgcn_exp2f(raise);
  }
}

// Both kinds of parts in one launch, spread evenly among each other: the
// prefix's multiply while the caches' are read (128 sequences behind 16,384
// keys: 157 us and 44 us one after the other, 173 us together).
template <typename T, int D>
__global__ __launch_bounds__(kThreads, (Prefix<T, D>::kWaves)) void
shared_prefix_parts(StepArgs a) {
  __shared__ __align__(1024) char lds[Prefix<T, D>::kBytes];
  __shared__ Totals found;
  __shared__ int verdict;
  const int64_t all = gridDim.x, prefix = a.wide_items;
  const int64_t before = blockIdx.x * prefix / all;
  if ((blockIdx.x + (int64_t)1) * prefix / all > before)
    // (the row tiles of a chunk next to each other on one XCD)
    prefix_part<T, D>(a, xcd_contiguous(before, prefix), lds, &verdict);
  else
    cache_part<T, D, false>(a, blockIdx.x - before, lds, found);
}

// Joins the parts of a query head's softmax: one workgroup for each, whose
// eight half waves take the parts in turn, DIM / 32 consecutive elements a
// lane, and are joined in LDS.  A launch and two trips: 16 parts of 4 sequences
// and 32 heads 4.4 us, 128 sequences' 8.4 us.
template <typename T, int DIM>
__global__ __launch_bounds__(kThreads) void window_cache_join(StepArgs a) {
  constexpr int N = DIM / 32, kHalves = kThreads / 32;
  __shared__ float outs[kHalves][DIM], tops[kHalves], totals[kHalves];
  const int seq = (int)(blockIdx.x / a.query_heads);
  const int head = (int)(blockIdx.x % a.query_heads);
  const int hk = head / a.group, row = head % a.group;
  const Visible see(a, seq);
  const int own = see.count == 0 ? 0 : (see.count - 1) / a.chunk + 1;
  const int parts = own + a.prefix_parts;
  const int half = threadIdx.x / 32, c = (threadIdx.x % 32) * N;
  float top = -kInf, l = 0.0f, o[N] = {};
#pragma unroll 4
  for (int i = half; i < parts; i += kHalves) {
    // row of part i in the buffers of sums and statistics
    const int64_t r =
        i < own ? (((int64_t)seq * a.key_heads + hk) * a.parts + i) * a.rows + row
                : ((int64_t)hk * a.prefix_parts + i - own) * a.prefix_rows +
                      (int64_t)seq * a.group + row;
    const float *sums = (i < own ? a.sums : a.prefix_sums) + r * DIM + c;
    const float *stats = (i < own ? a.stats : a.prefix_stats) + r * 2;
    const float m = stats[0], to = fmaxf(top, m);
    const float by = top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to);
    const float add = m == to ? 1.0f : __builtin_amdgcn_exp2f(m - to);
    const float weight = stats[1] * a.lower * add;
    top = to;
    l = fmaf(l, by, weight);
#pragma unroll
    for (int e = 0; e < N; ++e)
      o[e] = fmaf(sums[e], weight, o[e] * by);
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    outs[half][c + e] = o[e];
  if (threadIdx.x % 32 == 0) {
    tops[half] = top;
    totals[half] = l;
  }
  __syncthreads();
  if (threadIdx.x >= a.d)
    return;
  top = tops[0];
#pragma unroll
  for (int i = 1; i < kHalves; ++i)
    top = fmaxf(top, tops[i]);
  float x = 0.0f;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < kHalves; ++i) {
    const float by =
        tops[i] == top ? 1.0f : __builtin_amdgcn_exp2f(tops[i] - top);
    l = fmaf(totals[i], by, l);
    x = fmaf(outs[i][threadIdx.x], by, x);
  }
  stv(static_cast<T *>(a.output) + seq * a.output_token +
          head * a.output_head + threadIdx.x,
      top == -kInf ? 0.0f : x * (1.0f / l));
}

// ---- host ------------------------------------------------------------------------

// How a call is cut into parts.
struct Plan {
  int64_t chunk, parts, rows, prefix_chunk, prefix_parts, prefix_rows;
  bool wide; // the prefix by shared_prefix_parts
  int64_t sums, stats, prefix_sums, prefix_stats; // floats
  int64_t bytes() const {
    return 4 * (sums + stats + prefix_sums + prefix_stats);
  }
};

// Query rows of a key head (of all sequences) past which a prefix goes through
// tiles of 128 of them instead of 16.  8 key heads, caches of up to 256 keys
// behind the prefix, parts of 128 / of 16 rows, us:
//   rows, prefix      bf16, d = 128   bf16, 64      fp32, 64      fp32, 128
//    32,  1000        12.3 / 12.6     10.1 /  9.8   24.9 / 12.5    41.6 /  19.7
//    64,  1000        13.0 / 13.2     10.5 / 10.3   25.7 / 13.3    43.6 /  21.4
//    96,  1000        14.4 / 16.3     11.2 / 12.0   26.7 / 16.6    45.0 /  36.1
//   256,  1000        25.6 / 28.4     16.3 / 17.7   34.9 / 28.5    78.0 /  68.4
//    32,  8192        17.4 / 21.5     12.4 / 14.2   29.0 / 21.5    80.8 /  51.9
//    64,  8192        19.4 / 31.2     14.6 / 19.6   41.8 / 31.7    83.3 /  81.9
//    96,  8192        22.1 / 39.6     15.6 / 23.8   43.5 / 40.8    86.1 / 108.2
//   256,  8192        38.8 / 67.7     22.0 / 35.7   55.6 / 71.8   155.7 / 219.4
// One number for all: bf16 behind a long prefix would gain from 16 rows on, fp32
// behind a short one only past 256.
constexpr int64_t kWideRows = 64;

Plan plan(int64_t sequences, int64_t capacity, int64_t query_heads,
          int64_t key_heads, int64_t d, int64_t window, int64_t sinks,
          int64_t prefix_tokens) {
  Plan p{};
  const int64_t dim = d <= 64 ? 64 : 128, group = query_heads / key_heads;
  p.rows = sw::ceil_div(group, kRows) * kRows;
  const int64_t visible =
      window >= capacity || sinks >= capacity - window ? capacity
                                                       : window + sinks;
  auto cut = [](int64_t n, int64_t units, int64_t want, int64_t least,
                int64_t step) {
    const int64_t parts = std::max<int64_t>(1, sw::ceil_div(want, units));
    const int64_t chunk = std::max(least, sw::ceil_div(n, parts));
    return std::min<int64_t>(sw::ceil_div(chunk, step) * step, 1 << 30);
  };
  // Few keys are one part: a second one and the join of both cost more (32 query
  // heads over 8, bf16 of 128, one part / two, us: 300 keys of one sequence
  // 11.0 / 11.9, of 32 sequences 11.4 / 16.2; 512 keys 13.7 / 12.1 and
  // 16.5 / 17.0; 700 keys 17.4 / 12.1 and 20.8 / 20.4; fp32 of 64: 300 keys
  // 12.2 / 12.2 and 12.7 / 17.4, 512 keys 15.5 / 12.4 and 18.8 / 18.1, 700 keys
  // 20.4 / 12.5 and 24.9 / 22.2).
  // The cut is by the keys that there is room for, which the host knows: much
  // more room than keys makes few and long parts.  64 sequences of 4096 keys take
  // 194 us with room for 4096 to 131,072; one takes 12.8, and 18.9 with room for
  // 32,768, 55.9 for 131,072; four 19.7, 56.7 and 100.4.
  p.chunk = visible <= 512
                ? 512
                : cut(visible, sequences * key_heads * (p.rows / kRows), 512,
                      256, 128);
  p.parts = std::max<int64_t>(1, sw::ceil_div(visible, p.chunk));
  if (prefix_tokens > 0) {
    const int64_t rows = sequences * group;
    p.wide = rows > kWideRows;
    const int64_t step = p.wide ? kPrefixRows : kRows;
    p.prefix_rows = sw::ceil_div(rows, step) * step;
    p.prefix_chunk = cut(prefix_tokens, key_heads * (p.prefix_rows / step),
                         p.wide ? 256 : 1024, 256, 128);
    p.prefix_parts = sw::ceil_div(prefix_tokens, p.prefix_chunk);
  }
  if (p.parts == 1 && p.prefix_parts == 0)
    return p;
  const int64_t all = sequences * key_heads * p.parts * p.rows;
  const int64_t shared = key_heads * p.prefix_parts * p.prefix_rows;
  p.sums = all * dim;
  p.stats = all * 2;
  p.prefix_sums = shared * dim;
  p.prefix_stats = shared * 2;
  return p;
}

int check_sizes(int64_t sequences, int64_t pages, int64_t page_size,
                int64_t table_width, int64_t query_heads, int64_t key_heads,
                int64_t d, int64_t window, int64_t sinks,
                int64_t prefix_tokens, float alpha) {
  if (sequences < 0 || pages < 0 || page_size < 1 || table_width < 1 ||
      prefix_tokens < 0 || sequences > (1 << 24) || pages > sw::kMostTokens ||
      page_size > sw::kMostTokens || prefix_tokens > sw::kMostTokens ||
      table_width > sw::kMostTokens / page_size)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "expected up to 2^24 sequences, and pages of a size and a "
                    "table of a width that hold up to 2^30 keys, but got "
                    "%lld, %lld, %lld, %lld and a prefix of %lld",
                    (long long)sequences, (long long)pages,
                    (long long)page_size, (long long)table_width,
                    (long long)prefix_tokens);
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

int check_pages(const char *name, const void *p, int64_t page, int64_t token,
                int64_t head, int64_t d, int64_t elem, int64_t pages,
                int64_t heads) {
  if (pages > 0 && (page < 0 || page > sw::kMostStride))
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "%s page stride must be 0 to 2^40, but got %lld", name,
                    (long long)page);
  if (int rc = check_operand(name, p, {token, head}, d, elem, false, pages,
                             heads))
    return rc;
  if (pages > 0 && page * elem % 16 != 0)
    return sw::fail(SW_ERR_INVALID_ARGUMENT,
                    "%s must be 16-byte aligned, its strides included", name);
  return SW_OK;
}

template <typename T>
int step_entry(const int32_t *key_lengths, const int32_t *page_table,
               const T *query, const T *prefix_key, const T *prefix_value,
               const T *key_cache, const T *value_cache, T *output,
               int64_t sequences, int64_t prefix_tokens, int64_t pages,
               int64_t page_size, int64_t table_width, int64_t query_heads,
               int64_t key_heads, int64_t d, const int64_t *strides,
               int64_t window, int64_t sinks, float alpha, void *workspace,
               int64_t workspace_bytes, void *stream, const char *what) {
  sw::clear_error();
  if (!page_table)
    table_width = 1;
  if (int rc = check_sizes(sequences, pages, page_size, table_width,
                           query_heads, key_heads, d, window, sinks,
                           prefix_tokens, alpha))
    return rc;
  if (!page_table && pages < sequences)
    return sw::fail(SW_ERR_INVALID_SHAPE,
                    "without a page table every sequence needs its page, but "
                    "got %lld pages for %lld sequences", (long long)pages,
                    (long long)sequences);
  if (sequences > 0 && !key_lengths)
    return sw::fail(SW_ERR_INVALID_ARGUMENT, "key lengths pointer is null");
  if (int rc = sw::check_value_alignment(4, {key_lengths, page_table}))
    return rc;
  const int64_t row = key_heads * d;
  const int64_t packed[14] = {
      query_heads * d, d, query_heads * d, d, page_size * row, row, d,
      page_size * row, row, d, row, d, row, d};
  const int64_t *s = strides ? strides : packed;
  if (int rc = check_operand("query", query, {s[0], s[1]}, d, sizeof(T), false,
                             sequences, query_heads))
    return rc;
  if (int rc = check_operand("output", output, {s[2], s[3]}, d, sizeof(T), true,
                             sequences, query_heads))
    return rc;
  if (int rc = check_pages("key cache", key_cache, s[4], s[5], s[6], d,
                           sizeof(T), pages, key_heads))
    return rc;
  if (int rc = check_pages("value cache", value_cache, s[7], s[8], s[9], d,
                           sizeof(T), pages, key_heads))
    return rc;
  StepArgs a{};
  if (prefix_tokens > 0) {
    // (only the shared-prefix entry points have these strides)
    if (int rc = check_operand("prefix key", prefix_key, {s[10], s[11]}, d,
                               sizeof(T), false, prefix_tokens, key_heads))
      return rc;
    if (int rc = check_operand("prefix value", prefix_value, {s[12], s[13]}, d,
                               sizeof(T), false, prefix_tokens, key_heads))
      return rc;
    a.prefix = {prefix_key, prefix_value, 0, s[10], s[11], 0, s[12], s[13]};
  }
  if (sequences == 0)
    return SW_OK;
  const Plan p = plan(sequences, page_size * table_width, query_heads,
                      key_heads, d, window, sinks, prefix_tokens);
  if (p.bytes() > 0 && (!workspace || !sw::aligned16(workspace) ||
                        workspace_bytes < p.bytes()))
    return sw::fail(SW_ERR_INVALID_ARGUMENT,
                    "%s needs a 16-byte aligned workspace of %lld bytes", what,
                    (long long)p.bytes());
  a.lengths = key_lengths;
  a.table = page_table;
  a.query = query;
  a.output = output;
  a.cache = {key_cache, value_cache, s[4], s[5], s[6], s[7], s[8], s[9]};
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
  a.prefix_tokens = (int)prefix_tokens;
  a.alpha = alpha;
  a.chunk = (int)p.chunk;
  a.parts = (int)p.parts;
  a.rows = (int)p.rows;
  a.prefix_chunk = (int)p.prefix_chunk;
  a.prefix_parts = (int)p.prefix_parts;
  a.prefix_rows = (int)p.prefix_rows;
  a.lower = std::ldexp(
      1.0f, -(int)std::ceil(std::log2((double)(p.chunk * p.parts +
                                               prefix_tokens))) - 1);
  a.sums = static_cast<float *>(workspace);
  a.stats = a.sums + p.sums;
  a.prefix_sums = a.stats + p.stats;
  a.prefix_stats = a.prefix_sums + p.prefix_sums;
  a.prefix_items = p.wide ? 0
                          : key_heads * (p.prefix_rows / kRows) * p.prefix_parts;
  a.wide_items =
      p.wide ? key_heads * (p.prefix_rows / kPrefixRows) * p.prefix_parts : 0;
  const int64_t grid = a.prefix_items + a.wide_items +
                       sequences * key_heads * (p.rows / kRows) * p.parts;
  const int64_t join = sequences * query_heads;
  if (int rc = sw::check_flat_grid(std::max(grid, join), kThreads, what))
    return rc;
  const hipStream_t st = sw::as_stream(stream);
  const dim3 g((unsigned)grid);
  if (p.wide && d <= 64)
    shared_prefix_parts<T, 64><<<g, kThreads, 0, st>>>(a);
  else if (p.wide)
    shared_prefix_parts<T, 128><<<g, kThreads, 0, st>>>(a);
  else if (d <= 64)
    window_cache_parts<T, 64><<<g, kThreads, 0, st>>>(a);
  else
    window_cache_parts<T, 128><<<g, kThreads, 0, st>>>(a);
  if (int rc = sw::launch_check(what))
    return rc;
  if (p.parts == 1 && p.prefix_parts == 0)
    return SW_OK;
  if (d <= 64)
    window_cache_join<T, 64><<<dim3((unsigned)join), kThreads, 0, st>>>(a);
  else
    window_cache_join<T, 128><<<dim3((unsigned)join), kThreads, 0, st>>>(a);
  return sw::launch_check(what);
}

template <typename T>
int decode_entry(const int32_t *key_lengths, const int32_t *page_table,
                 const T *query, const T *key_cache, const T *value_cache,
                 T *output, int64_t sequences, int64_t pages,
                 int64_t page_size, int64_t table_width, int64_t query_heads,
                 int64_t key_heads, int64_t d, const int64_t *strides,
                 int64_t window, int64_t sinks, float alpha, void *workspace,
                 int64_t workspace_bytes, void *stream) {
  return step_entry<T>(key_lengths, page_table, query, nullptr, nullptr,
                       key_cache, value_cache, output, sequences, 0, pages,
                       page_size, table_width, query_heads, key_heads, d,
                       strides, window, sinks, alpha, workspace,
                       workspace_bytes, stream, "window attention decode");
}

template <typename T>
int prefix_entry(const int32_t *key_lengths, const int32_t *page_table,
                 const T *query, const T *prefix_key, const T *prefix_value,
                 const T *key_cache, const T *value_cache, T *output,
                 int64_t sequences, int64_t prefix_tokens, int64_t pages,
                 int64_t page_size, int64_t table_width, int64_t query_heads,
                 int64_t key_heads, int64_t d, const int64_t *strides,
                 float alpha, void *workspace, int64_t workspace_bytes,
                 void *stream) {
  return step_entry<T>(key_lengths, page_table, query, prefix_key,
                       prefix_value, key_cache, value_cache, output, sequences,
                       prefix_tokens, pages, page_size, table_width,
                       query_heads, key_heads, d, strides, sw::kMostTokens, 0,
                       alpha, workspace, workspace_bytes, stream,
                       "shared prefix attention");
}

} // namespace

extern "C" int64_t sw_window_attention_decode_workspace_bytes(
    int64_t sequences, int64_t page_size, int64_t table_width,
    int64_t query_heads, int64_t key_heads, int64_t d, int64_t window,
    int64_t sinks) {
  if (sequences == 0 ||
      check_sizes(sequences, 0, page_size, table_width, query_heads, key_heads,
                  d, window, sinks, 0, 0.0f) != SW_OK)
    return 0;
  return plan(sequences, page_size * table_width, query_heads, key_heads, d,
              window, sinks, 0).bytes();
}

extern "C" int64_t sw_shared_prefix_attention_workspace_bytes(
    int64_t sequences, int64_t prefix_tokens, int64_t page_size,
    int64_t table_width, int64_t query_heads, int64_t key_heads, int64_t d) {
  if (sequences == 0 ||
      check_sizes(sequences, 0, page_size, table_width, query_heads, key_heads,
                  d, 1, 0, prefix_tokens, 0.0f) != SW_OK)
    return 0;
  return plan(sequences, page_size * table_width, query_heads, key_heads, d,
              sw::kMostTokens, 0, prefix_tokens).bytes();
}

extern "C" int sw_window_attention_decode_f32(
    const int32_t *key_lengths, const int32_t *page_table, const float *query,
    const float *key_cache, const float *value_cache, float *output,
    int64_t sequences, int64_t pages, int64_t page_size, int64_t table_width,
    int64_t query_heads, int64_t key_heads, int64_t d, const int64_t *strides,
    int64_t window, int64_t sinks, float alpha, void *workspace,
    int64_t workspace_bytes, void *stream) {
  return decode_entry<float>(key_lengths, page_table, query, key_cache,
                             value_cache, output, sequences, pages, page_size,
                             table_width, query_heads, key_heads, d, strides,
                             window, sinks, alpha, workspace, workspace_bytes,
                             stream);
}

extern "C" int sw_window_attention_decode_bf16(
    const int32_t *key_lengths, const int32_t *page_table,
    const uint16_t *query, const uint16_t *key_cache,
    const uint16_t *value_cache, uint16_t *output, int64_t sequences,
    int64_t pages, int64_t page_size, int64_t table_width,
    int64_t query_heads, int64_t key_heads, int64_t d, const int64_t *strides,
    int64_t window, int64_t sinks, float alpha, void *workspace,
    int64_t workspace_bytes, void *stream) {
  return decode_entry<uint16_t>(key_lengths, page_table, query, key_cache,
                                value_cache, output, sequences, pages,
                                page_size, table_width, query_heads, key_heads,
                                d, strides, window, sinks, alpha, workspace,
                                workspace_bytes, stream);
}

extern "C" int sw_shared_prefix_attention_f32(
    const int32_t *key_lengths, const int32_t *page_table, const float *query,
    const float *prefix_key, const float *prefix_value,
    const float *key_cache, const float *value_cache, float *output,
    int64_t sequences, int64_t prefix_tokens, int64_t pages,
    int64_t page_size, int64_t table_width, int64_t query_heads,
    int64_t key_heads, int64_t d, const int64_t *strides, float alpha,
    void *workspace, int64_t workspace_bytes, void *stream) {
  return prefix_entry<float>(key_lengths, page_table, query, prefix_key,
                             prefix_value, key_cache, value_cache, output,
                             sequences, prefix_tokens, pages, page_size,
                             table_width, query_heads, key_heads, d, strides,
                             alpha, workspace, workspace_bytes, stream);
}

extern "C" int sw_shared_prefix_attention_bf16(
    const int32_t *key_lengths, const int32_t *page_table,
    const uint16_t *query, const uint16_t *prefix_key,
    const uint16_t *prefix_value, const uint16_t *key_cache,
    const uint16_t *value_cache, uint16_t *output, int64_t sequences,
    int64_t prefix_tokens, int64_t pages, int64_t page_size,
    int64_t table_width, int64_t query_heads, int64_t key_heads, int64_t d,
    const int64_t *strides, float alpha, void *workspace,
    int64_t workspace_bytes, void *stream) {
  return prefix_entry<uint16_t>(key_lengths, page_table, query, prefix_key,
                                prefix_value, key_cache, value_cache, output,
                                sequences, prefix_tokens, pages, page_size,
                                table_width, query_heads, key_heads, d,
                                strides, alpha, workspace, workspace_bytes,
                                stream);
}
