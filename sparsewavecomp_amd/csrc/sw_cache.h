// What the kernels of single queries against a key-value cache share, of bf16 and
// fp32 values and of 4-bit codes: which keys a query sees, what a workgroup
// leaves of the keys it took, and the host's checks.
//
// Where several workgroups take a sequence's keys each leaves, of its part c of
// them, the maximum m_c, the sum l_c and the mean o_c, and they are joined:
//   m = max m_c,  w_c = l_c 2^(m_c - m),  l = sum w_c,  o = sum o_c w_c / l.
// Means and not sums of values, which fp32 may not hold where their mean is
// finite: those stay within a part, which sees whether they did.
#pragma once

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

struct Cache {
  const void *key, *value;
  int64_t key_page, key_token, key_head; // strides in elements
  int64_t value_page, value_token, value_head;
};

// (The prefix, `dim` and the parts' numbers and rows are sw_cache_attention.hip's
// alone.)
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
struct Totals {
  float top[4][kRows], sum[4][kRows], raise[4][kRows];
};

// The four waves' results of one part of the keys, joined in LDS and written:
// as the output where the part is the `only` one, else to `sums` and `stats`.
// acc: o[column][d] of a wave, which it leaves in its own WAVE_BYTES of `lds`;
// top, sum and raise: of column l % 16.  Columns ROWS apart are one row's, of
// different keys.
template <typename T, int D, int WAVE_BYTES, int ROWS = kRows>
__device__ __forceinline__ void
store_part(const StepArgs &a, char *lds, Totals &found, float top, float sum,
           float raise, const v4f (&acc)[D / 16], int rows, bool only, int seq,
           int hk, int first_row, float *sums, float *stats) {
  const int lane = lane_id(), g = lane >> 4, wave = wave_in_group();
  if (g == 0) {
    found.top[wave][lane] = top;
    found.sum[wave][lane] = sum;
    found.raise[wave][lane] = raise;
  }
  // o[column][d] of each wave, in its own part of LDS
#pragma unroll
  for (int b = 0; b < D / 16; ++b)
    lds_write(lds_address(lds) + wave * WAVE_BYTES +
                  ((lane & 15) * D + 16 * b + 4 * g) * 4, acc[b]);
  __syncthreads();
  constexpr int kParts = 4 * (kRows / ROWS); // of a row: wave i % 4, column r + ..
  for (int x = threadIdx.x; x < ROWS * D / 4; x += kThreads) {
    const int r = x / (D / 4), c = x % (D / 4) * 4;
    if (r >= rows)
      break;
    float m = found.top[0][r], most = found.raise[0][r];
#pragma unroll
    for (int i = 1; i < kParts; ++i) {
      m = fmaxf(m, found.top[i % 4][r + i / 4 * ROWS]);
      most = fmaxf(most, found.raise[i % 4][r + i / 4 * ROWS]);
    }
    // (as many sums that are finite have a finite sum)
    most += kRows / ROWS == 1 ? 3.0f : 5.0f;
    float l = 0.0f;
    v4f o = {};
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int w = i % 4, column = r + i / 4 * ROWS;
      float by = found.top[w][column] == -kInf
                     ? 0.0f
                     : __builtin_amdgcn_exp2f(found.top[w][column] - m);
      by *= __builtin_amdgcn_exp2f(found.raise[w][column] - most);
      const v4f y = lds_read<v4f>(
          lds_address(lds) + w * WAVE_BYTES + (column * D + c) * 4, 0);
      l = fmaf(found.sum[w][column], by, l);
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

// A row of a part.
struct PartRow {
  const float *sums, *stats;
};

// ---- host ------------------------------------------------------------------------

// The keys that a query sees at most.
inline int64_t most_visible(int64_t capacity, int64_t window, int64_t sinks) {
  return window >= capacity || sinks >= capacity - window ? capacity
                                                          : window + sinks;
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

} // namespace
