// Attention of one query for each sequence against a key-value cache of 4-bit
// codes, over a sliding window with sinks.
//
// The arithmetic of the cache attention over bf16 values (sw_cache_attention.hip):
// a code times its block's scale is a bf16 number, so the bf16 matrix cores
// multiply with it exactly, and fp32 queries, cut into three bf16 parts, and
// probabilities lose nothing either.  A key and its value take 17/16 d bytes for
// 4 G d operations of the G query heads that share them: 3.75 times fewer bytes
// than in bf16, for the same products, exponentials and conversions besides.
//
// Memory bounds long batches: 64 sequences of up to 20,000 keys, 32 query heads
// over 8 of 128, bf16, 887 MB, take 154 us in the kernel and 5 in the join (the
// medians of 22; at best 144 and 4), 5.6 TB/s with both; the same loads alone,
// streamed, take 134.  The matrix cores are busy for 25 % of it, vector instructions
// for 44 %.  Heads of 64 and 32 are bound by the instructions of a tile, which are
// not many fewer for its fewer bytes: 64 sequences of up to 20,000, 16 heads over 4
// of 64, 57 us, 3.9 TB/s.  In fp32 (5 sequences, windows of 65,544 keys, 12 heads
// over 4 of 96, 104 MB: 36 and 5 us) three parts of queries and of probabilities
// are three times the products.  A short call is its chain of trips (length, page,
// key) and the join's, and so is each sequence's part of a batch of short ones: 64
// of up to 1,024 keys, 32 heads over 8 of 128, take 19 us, their bytes 6.5.
#include "sw_cache.h"
#include "sw_fp4.h"

namespace {

// how many powers of two a part's maximum may lag
constexpr float kLag = 8.0f;

struct Scales {
  const uint8_t *key, *value;
  int64_t key_page, key_token, key_head; // strides in bytes
  int64_t value_page, value_token, value_head;
};

struct Fp4StepArgs {
  StepArgs s; // (its cache: the codes, strides in bytes)
  Scales scales;
  Divisor page_size;
  // A unit is `block` query rows (8 or 16) of a key head, for all sequences.  Its
  // tiles are split evenly among `shares` workgroups, each taking `least` at
  // least.  0 shares: a workgroup for each sequence of a unit, which has `least`
  // tiles at most.
  int units, shares, least, block;
};

// The tiles of kTile keys, from multiples of it on, that hold the keys that a
// sequence's query sees: the sinks' that lie before the window's first one, and
// the window's.
struct Tiles : Visible {
  using Visible::Visible;
  __device__ __forceinline__ int end() const { return start + count - lead; }
  __device__ __forceinline__ bool sees(int j) const {
    return (j < lead || j >= start) && j < end();
  }
  __device__ __forceinline__ int sink_tiles() const {
    const int sinks = (lead + kTile - 1) / kTile, first = start / kTile;
    return sinks < first ? sinks : first;
  }
  __device__ __forceinline__ int tiles() const {
    return count == 0 ? 0
                      : sink_tiles() + (end() + kTile - 1) / kTile -
                            start / kTile;
  }
  __device__ __forceinline__ int first_key(int tile) const {
    const int sinks = sink_tiles();
    return kTile * (tile < sinks ? tile : tile - sinks + start / kTile);
  }
};
__device__ __forceinline__ int tiles_of(const StepArgs &a, int sequence) {
  return Tiles(a, sequence).tiles();
}

// The same of a sequence that is wave-uniform, in scalar registers.
__device__ __forceinline__ Tiles uniform_tiles(const StepArgs &a,
                                               int sequence) {
  Tiles see(a, sequence);
  see.lead = __builtin_amdgcn_readfirstlane(see.lead);
  see.start = __builtin_amdgcn_readfirstlane(see.start);
  see.count = __builtin_amdgcn_readfirstlane(see.count);
  return see;
}

// The sum over this lane and those before it.
__device__ __forceinline__ int sum_to_lane(int v) {
  v += dpp_i<kRowShr1>(0, v);
  v += dpp_i<kRowShr2>(0, v);
  v += dpp_i<kRowShr4>(0, v);
  v += dpp_i<kRowShr8>(0, v);
  // (the last lane of rows 0 and 2 into rows 1 and 3, then of row 1 into both)
  v += dpp_i<kRowBcast15, 0xA>(0, v);
  v += dpp_i<kRowBcast31, 0xC>(0, v);
  return v;
}

// The tiles of up to 4096 sequences: lane l of a wave has those of number
// l each to l each + each - 1, the first HELD of them in registers (1, where that
// is all, or 4: with 8 for one sequence a call took 1.5 us longer, for 122 of up to
// 1,495 keys 21.8 us for 19.8).
template <int HELD> struct AllTiles {
  const StepArgs &a;
  int each, held[HELD];
  __device__ __forceinline__ explicit AllTiles(const StepArgs &args)
      : a(args), each(HELD == 1 ? 1 : (args.sequences + kWave - 1) / kWave) {
    load(held, 0);
  }
  __device__ __forceinline__ int of(int sequence, bool there = true) const {
    const int last = a.sequences - 1;
    const int tiles = tiles_of(a, sequence < last ? sequence : last);
    return there && sequence <= last ? tiles : 0;
  }
  // (their loads are on their way together)
  __device__ __forceinline__ void load(int (&n)[HELD], int from) const {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      n[i] = of(lane_id() * each + from + i, from + i < each);
  }
  // The sum of value(tiles) over this lane's first `end` ones; value(0) is 0.
  template <typename F>
  __device__ __forceinline__ int sum(int end, F value) const {
    int x = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      x += i < end ? value(held[i]) : 0;
    for (int from = HELD; from < end; from += HELD) {
      int n[HELD];
      load(n, from);
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        x += from + i < end ? value(n[i]) : 0;
    }
    return x;
  }
  template <typename F> __device__ __forceinline__ int sum(F value) const {
    return sum(each, value);
  }
};

// How a unit's tiles are split: `most` for a workgroup, and whether none takes
// those of two sequences (`whole`: a sequence's tiles are divided among its
// shares).  A second sequence costs a workgroup about as much as 8 tiles (4
// sequences of up to 8,192 keys 21.4 us, whole 19.2; 32 of up to 2,048 23.3 and
// 21.0; 64 of up to 20,000, over four key heads of 64, 56.5 and 58.2), so that
// shares may be longer by as much to keep them whole: by as little as does, where
// a wave has all sequences' tiles in registers.
struct Split {
  int most;
  bool whole;
  float by; // 1 / most
  template <int HELD>
  __device__ __forceinline__ Split(const Fp4StepArgs &args, int total,
                                   const AllTiles<HELD> &all) {
    constexpr int kSecond = 8;
    const int even = (total + args.shares - 1) / args.shares;
    const int fewest = even < args.least ? args.least : even;
    if (all.each <= HELD) {
      auto fits = [&](int n) __attribute__((always_inline)) {
        set(n);
        const int own = all.sum([&](int t) { return shares(t); });
        return __builtin_amdgcn_readlane(sum_to_lane(own), kWave - 1) <=
               args.shares;
      };
      int n = fewest + kSecond;
      whole = args.s.sequences < args.shares && fits(n);
      if (whole) {
        if (fits(fewest))
          n = fewest;
        else
          for (int step = kSecond / 2; step > 0; step /= 2)
            n -= fits(n - step) ? step : 0;
      }
      set(whole ? n : fewest);
    } else {
      const int apart = args.shares - args.s.sequences;
      const int more = apart > 0 ? (total + apart - 1) / apart : INT32_MAX;
      whole = more <= fewest + kSecond;
      set(whole && more > fewest ? more : fewest);
    }
  }
  __device__ __forceinline__ void set(int n) {
    most = n;
    by = __builtin_amdgcn_rcpf((float)n);
  }
  // Of a whole sequence: about tiles / most rounded up (in 32 bits, the same in
  // each wave that asks; at least 1 of a tile, and up to 4096 sequences no more in
  // all than exact ones could be).
  __device__ __forceinline__ int shares(int tiles) const {
    return (int)ceilf((float)tiles * by);
  }
};

// A workgroup's share of a unit's tiles: those from `from` on, of which sequence
// `seq` has the ones from `offset` on.  Up to 4096 sequences: a lane of a wave
// sums up to 64 of them, the sums are added up over the lanes, and then those of
// one lane.  What is summed are tiles, or where sequences stay whole their shares.
struct Share {
  int from, to, seq, offset;
};
template <int HELD>
__device__ __forceinline__ Share find_share(const Fp4StepArgs &args, int p) {
  const AllTiles<HELD> all(args.s);
  auto tiles = [](int n) { return n; };
  int own = all.sum(tiles);
  int sum = sum_to_lane(own);
  const int total = __builtin_amdgcn_readlane(sum, kWave - 1);
  const Split split(args, total, all);
  auto shares = [&](int n) { return split.shares(n); };
  Share s{0, 0, 0, 0};
  int first = p, end = total; // what is looked for, and of how many
  if (split.whole) {
    own = all.sum(shares);
    sum = sum_to_lane(own);
    end = __builtin_amdgcn_readlane(sum, kWave - 1);
  } else if (p > total / split.most) {
    return s; // (nothing is left)
  } else {
    first = p * split.most;
  }
  if (first >= end)
    return s;
  int at = __builtin_popcountll(ballot(sum <= first));
  s.seq = at * all.each;
  int offset = __builtin_amdgcn_readlane(sum - own, at);
  int held = all.held[0];
  if (all.each > 1) {
    held = lane_id() < all.each ? all.of(s.seq + lane_id()) : 0;
    own = split.whole ? shares(held) : held;
    sum = offset + sum_to_lane(own);
    at = __builtin_popcountll(ballot(lane_id() < all.each && sum <= first));
    s.seq += at;
    if (s.seq >= args.s.sequences) // (only if lengths change under the call)
      return s;
    offset = __builtin_amdgcn_readlane(sum - own, at);
  }
  if (split.whole) {
    const int n = __builtin_amdgcn_readlane(held, at);
    const int parts = n > 0 ? shares(n) : 1, i = p - offset;
    const int even = n / parts, longer = n - even * parts;
    s.from = i * even + (i < longer ? i : longer);
    s.to = s.from + even + (i < longer ? 1 : 0);
  } else {
    s.from = first;
    s.to = total - first < split.most ? total : first + split.most;
    s.offset = offset;
  }
  return s;
}

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

// Four probabilities as the sum of two bf16 parts, to 2^-15 of each, or of three,
// to 2^-23: what their upper halves hold, and the rest of it, at the end rounded.
// The rest of one that is not zero is at least 2^-126, so that an infinity of a
// value meets no zero that stands for it.
template <int N>
__device__ __forceinline__ void weight_parts(const float *x, v2u (&part)[N]) {
  float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    part[i] = v2u{__builtin_amdgcn_perm(__float_as_uint(r[1]),
                                        __float_as_uint(r[0]), 0x07060302u),
                  __builtin_amdgcn_perm(__float_as_uint(r[3]),
                                        __float_as_uint(r[2]), 0x07060302u)};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r[e] = __builtin_amdgcn_fmed3f(
          r[e] - __uint_as_float(__float_as_uint(r[e]) & 0xFFFF0000u), 0x1p-126f,
          r[e]);
  }
  part[N - 1] = v2u{cvt_pk_bf16(r[0], r[1]), cvt_pk_bf16(r[2], r[3])};
}

// Rows of 16-bit values of a wave's LDS, in chunks of 16 bytes; chunk c of row r
// lies at place c ^ swizzle(r).  Free of bank conflicts: a write of one chunk of
// eight consecutive rows (32 banks of 4 bytes; with the swizzle of RowTile such
// writes took twice as long), and half a wave's transposing load, two chunks of
// eight rows (64 banks).
template <int D> struct ValueTile {
  static constexpr int kPitch = 2 * D;
  static constexpr int kBytes = 32 * kPitch;
  __device__ static __forceinline__ int place(int row, int chunk) {
    const int swizzle =
        D > 64   ? (row & 4) << 1 | (row & 1) << 2 | (row & 2) | (row >> 2 & 1)
        : D > 32 ? (row & 2) << 1 | (row >> 1 & 2) | (row & 1)
                 : row >> 1 & 3;
    return row * kPitch + ((chunk ^ swizzle) << 4);
  }
};

// Of a SIMD's waves the one with most left to do goes first.  Left to themselves
// the oldest does: the three workgroups of a compute unit, which have the same to
// do, ended after 111, 124 and 142 us and left it half idle (124, 132 and 141 so,
// and in all 166.6 us -> 163.1; heads of 64 59.7 -> 57.1).  Later thresholds and quarters
// balance less.
__device__ __forceinline__ void go_first(int all, int left) {
  if (left > all / 2)
    __builtin_amdgcn_s_setprio(3);
  else if (left > all / 4)
    __builtin_amdgcn_s_setprio(2);
  else if (left > all / 8)
    __builtin_amdgcn_s_setprio(1);
  else
    __builtin_amdgcn_s_setprio(0);
}

// One share of a unit's tiles, a tile a wave at a time, part by part (a part:
// the share's tiles of one sequence).  Lane l holds a quarter (l / 16) of key
// l % 16 of each of the tile's runs of 16 keys, whose codes are one load for
// d = 128; quarter g of step st is elements D / 4 g + 8 st + i of the products'
// K index, in the queries too.  Values go through LDS as bf16, to be read across
// their rows.
//
// A run of 16 keys lies in one page wherever a page holds a multiple of 16: its
// addresses are then scalar ones plus a lane's constant offset.  Runs that cross
// a page's end take each lane's own.  The pages of a wave's next runs are found
// 64 at once, one by each lane.  (The batch above: 413 us with each lane's
// addresses for each key, 310 so, 185 with even shares and the queries' fragments
// in LDS instead of registers, 167 with the next tile's loads under way.  The next
// tile's scores before this one's values: 339.)
//
// Up to 8 query rows (ROWS) have the 16 columns of a product twice, each half for
// the scores of one of the tile's two runs, so that a lane has 4 scores instead of
// 8, half of them of rows that are not there.  A half's probabilities are masked
// out where the other run's values are multiplied; each column keeps a maximum and
// sums of its own, joined like a part's at the end.  (171 us for 175; 8 heads a key
// head 156 for 157.)  Where that leaves sums that are not finite (a zero of these
// masks times an infinity may be why) each run is multiplied by itself.
//
// STREAM: the codes pass by the caches, where no other workgroup reads them: up to
// 16 rows (166 us, 174 through them; 16 heads a key head 91 and 99); with 32, whose
// two workgroups read the same keys, 168 past them and 156 through them.
template <typename T, int D> struct Fp4Parts {
  using Tile = ValueTile<D>;
  static constexpr int kWaveBytes =
      Tile::kBytes > kRows * D * 4 ? Tile::kBytes : kRows * D * 4;
  static constexpr int kBytes = 4 * kWaveBytes;
  // waves of a SIMD (heads of 32: 46 sequences of up to 28,000 keys, 24 over 8, bf16
  // 88 us with 5, 98 with 4, and 92 as heads of 64; fp32 spills with 5)
  static constexpr int kWaves = D > 64                        ? 3
                                : D > 32 || sizeof(T) == 4 ? 4
                                                              : 5;
};

template <typename T, int D, int ROWS, bool STREAM>
__global__ __launch_bounds__(kThreads, (Fp4Parts<T, D>::kWaves)) void
fp4_cache_parts(Fp4StepArgs args) {
  using F = Fp4Parts<T, D>;
  using Tile = typename F::Tile;
  constexpr int kSteps = D / 32;  // products along d
  constexpr int kBlocks = D / 16; // output rows of 16
  constexpr int kWords = D / 32;  // words of codes of a lane's quarter row
  constexpr bool kHalves = ROWS == 8;
  constexpr int kSets = kHalves ? 1 : 2; // of 4 scores a lane
  __shared__ __align__(1024) char lds[F::kBytes];
  // the queries' fragments, [part][step][lane], which all waves read
  __shared__ v4u queries[kQueryParts<T> * kSteps * kWave];
  __shared__ Totals found;
  const StepArgs &a = args.s;

  const int lane = lane_id(), g = lane >> 4, wave = wave_in_group();
  const int row_of = lane & 15; // key of a run, column of a product
  // (neighbours take the units in turn, starting with another one each time: an
  // XCD, which gets every eighth workgroup, does not keep to one head's rows)
  const int number = (int)(blockIdx.x / args.units);
  const int unit = (int)((blockIdx.x + number) % args.units);
  const int blocks = (a.group + ROWS - 1) / ROWS; // of rows, of a key head
  const int hk = unit / blocks;
  const int first_row = (unit - hk * blocks) * ROWS;
  const int rows = a.group - first_row < ROWS ? a.group - first_row : ROWS;
  const bool live = row_of % ROWS < rows;
  Share my{0, 0, number, 0};
  int extent = args.least; // the share's tiles
  bool begun = false; // whether a part of the share is done
  if (args.shares != 0) {
    // (one wave for all: 122 sequences of up to 1,495 keys 21.8 us, 28.5 with each)
    __shared__ Share share;
    if (wave == 0) {
      my = a.sequences <= kWave ? find_share<1>(args, number)
                                : find_share<4>(args, number);
      if (lane == 0)
        share = my;
    }
    __syncthreads();
    my.from = __builtin_amdgcn_readfirstlane(share.from);
    my.to = __builtin_amdgcn_readfirstlane(share.to);
    my.seq = __builtin_amdgcn_readfirstlane(share.seq);
    my.offset = __builtin_amdgcn_readfirstlane(share.offset);
    if (my.from == my.to)
      return;
    extent = my.to - my.from;
  }
  const bool none = a.alpha == 0.0f;
  const float scale = __uint_as_float(__builtin_amdgcn_readfirstlane(
      __float_as_uint(none ? 1.0f : fabsf(a.alpha) * kLog2e)));

  // This lane's quarter of a row: codes, and the scale of its block.  Quarters
  // past d read the row's first one; the queries are zero there, and so is the
  // scale.
  const bool inside = D / 4 * g < a.d;
  const int code_at = inside ? D / 8 * g : 0, scale_at = inside ? D * g / 128 : 0;
  const Scales &sc = args.scales;
  const uint8_t *key_codes =
      static_cast<const uint8_t *>(a.cache.key) + hk * a.cache.key_head;
  const uint8_t *value_codes =
      static_cast<const uint8_t *>(a.cache.value) + hk * a.cache.value_head;
  const uint8_t *key_scales = sc.key + hk * sc.key_head;
  const uint8_t *value_scales = sc.value + hk * sc.value_head;
  // (a token stride is at most 2^23)
  uint32_t key_off = row_of * (uint32_t)a.cache.key_token + code_at;
  uint32_t value_off = row_of * (uint32_t)a.cache.value_token + code_at;
  uint32_t key_scale_off = row_of * (uint32_t)sc.key_token + scale_at;
  uint32_t value_scale_off = row_of * (uint32_t)sc.value_token + scale_at;

  // (of the sequence at hand, set below)
  int seq = my.seq, t0, t1;
  Tiles see = uniform_tiles(a, seq);
  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  struct Data {
    Words key[2], value[2];
    uint32_t key_scale[2], value_scale[2];
    uint32_t has[2]; // bit i: key i of the run is seen (wave-uniform)
  };
  // Of the wave's next tiles: lane l has run l % 2 of tile l / 2.
  enum { kNone, kWhole, kCut };
  struct Runs {
    int state; // whether it lies in one page, crosses a page's end, or neither
    int64_t key, value, key_scale, value_scale; // where its rows start
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
    const int tile = first + 4 * (lane / 2);
    const int key = see.first_key(tile) + 16 * (lane % 2);
    Runs r{kNone, 0, 0, 0, 0};
    if (tile < t1 && key < see.end()) {
      int slot;
      const int64_t page = page_of(key, slot);
      r.state = slot + 16 > a.page_size ? kCut : page < 0 ? kNone : kWhole;
      r.key = page * a.cache.key_page + slot * a.cache.key_token;
      r.value = page * a.cache.value_page + slot * a.cache.value_token;
      r.key_scale = page * sc.key_page + slot * sc.key_token;
      r.value_scale = page * sc.value_page + slot * sc.value_token;
    }
    return r;
  };
  // An address in scalar registers, to which a load adds a lane's offset.
  typedef const __attribute__((address_space(1))) uint8_t *Global;
  typedef const __attribute__((address_space(1))) Words *GlobalWords;
  auto scalar = [&](const uint8_t *p, int64_t at, int from)
                    __attribute__((always_inline)) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)at, from);
    const int hi = __builtin_amdgcn_readlane((int)(at >> 32), from);
    uint64_t address = (uint64_t)p + ((uint64_t)(uint32_t)hi << 32 | lo);
    asm("" : "+s"(address));
    return (Global)address;
  };
  auto codes = [](GlobalWords p) __attribute__((always_inline)) {
    if constexpr (STREAM)
      return __builtin_nontemporal_load(p);
    else
      return *p;
  };
  // tile k of those located, whose first key is `key`
  auto fetch = [&](Data &x, const Runs &r, int k, int key)
                   __attribute__((always_inline)) {
    // (32 bits, which the loads extend)
    asm volatile("" : "+v"(key_off), "+v"(value_off), "+v"(key_scale_off),
                 "+v"(value_scale_off));
#pragma unroll
    for (int b = 0; b < 2; ++b, key += 16) {
      const int from = 2 * k + b;
      const int state = __builtin_amdgcn_readlane(r.state, from);
      x.has[b] = 0;
      if (state == kWhole) {
        const Global kc = scalar(key_codes, r.key, from);
        const Global vc = scalar(value_codes, r.value, from);
        const Global ks = scalar(key_scales, r.key_scale, from);
        const Global vs = scalar(value_scales, r.value_scale, from);
        x.key[b] = codes((GlobalWords)(kc + key_off));
        x.key_scale[b] = ks[key_scale_off];
        x.value[b] = codes((GlobalWords)(vc + value_off));
        x.value_scale[b] = vs[value_scale_off];
        const bool all = (key + 16 <= see.lead || key >= see.start) &&
                         key + 16 <= see.end();
        x.has[b] = all ? 0xFFFFu
                       : (uint32_t)ballot(see.sees(key + row_of)) & 0xFFFFu;
      } else {
        x.key[b] = x.value[b] = Words{};
        x.key_scale[b] = x.value_scale[b] = 0;
        if (state == kCut) {
          int slot = 0, lane_row = row_of, code = code_at, block = scale_at;
          // (what this path needs is not held for it)
          asm volatile("" : "+v"(lane_row), "+v"(code), "+v"(block));
          int64_t page = -1;
          if (see.sees(key + lane_row))
            page = page_of(key + lane_row, slot);
          if (page >= 0) {
            x.key[b] = *reinterpret_cast<const Words *>(
                key_codes + page * a.cache.key_page +
                slot * a.cache.key_token + code);
            x.value[b] = *reinterpret_cast<const Words *>(
                value_codes + page * a.cache.value_page +
                slot * a.cache.value_token + code);
            x.key_scale[b] =
                key_scales[page * sc.key_page + slot * sc.key_token + block];
            x.value_scale[b] = value_scales[page * sc.value_page +
                                            slot * sc.value_token + block];
          }
          x.has[b] = (uint32_t)ballot(page >= 0) & 0xFFFFu;
        }
      }
    }
  };

  v4f acc[kBlocks], total; // total: the probabilities' sums, in all four
  float top;
  float lower = 1.0f; // of this lane's column: a factor of the probabilities
  const uint32_t own = lds_address(lds) + wave * F::kWaveBytes;
  // of a read across rows 4 g + .. and of a write: chunks differ by what the
  // swizzle leaves alone, rows 16 apart have the same
  uint32_t across = own + Tile::place(4 * g + (row_of >> 2), (lane & 3) >> 1) +
                    (lane & 1) * 8;
  uint32_t along = own + Tile::place(row_of, kWords * g);
  const uint32_t query_at = lds_address(queries) + lane * 16;
  const v4u ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

  auto compute = [&](Data &x, auto careful) __attribute__((always_inline)) {
    // whether a column's zeros for the other run meet none of its values, which
    // may be infinite
    constexpr bool kApart = kHalves && decltype(careful)::value;
    // (keeps the compiler from holding every address in a register)
    asm volatile("" : "+v"(across), "+v"(along));
    // element i of set s: of key 4 g + i of run s, or with halves of this
    // column's run
    v4f score[kSets];
    {
      v4f product[2] = {};
      float by[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
        by[b] = fp4_scale(inside ? x.key_scale[b] : 0u);
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        v4u q[kQueryParts<T>];
#pragma unroll
        for (int i = 0; i < kQueryParts<T>; ++i)
          q[i] = lds_read<v4u>(query_at, (i * kSteps + st) * kWave * 16);
        const v4u k[2] = {fp4_values(x.key[0][st], by[0]),
                          fp4_values(x.key[1][st], by[1])};
        // (the runs in turn: a product waits for the one before of its run)
#pragma unroll
        for (int i = kQueryParts<T> - 1; i >= 0; --i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            product[b] = mma16(k[b], q[i], product[b]);
      }
      if constexpr (kHalves) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          score[0][i] = row_of < ROWS ? product[0][i] : product[1][i];
      } else {
        score[0] = product[0];
        score[1] = product[1];
      }
    }
    if ((x.has[0] & x.has[1]) != 0xFFFFu) {
#pragma unroll
      for (int s = 0; s < kSets; ++s) {
        const uint32_t seen =
            (kHalves && row_of >= ROWS ? x.has[1] : x.has[s]) >> (4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(seen & (1u << i)))
            score[s][i] = -kInf;
      }
      // (what lies at a place that is not seen may be NaN)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        if (!(x.has[b] >> row_of & 1))
          x.value_scale[b] = 0;
    }
    float big = score[0][0];
#pragma unroll
    for (int i = 1; i < 4 * kSets; ++i)
      big = fmaxf(big, score[i / 4][i % 4]);
    big *= scale;
    // The maximum lags by up to 2^8: fewer sums are scaled anew, and a column's
    // four lanes only then compare theirs.
    if (ballot(big > top + kLag) != 0) {
      const float to = fmaxf(top, rows16_max(big));
      const float by = to == -kInf ? 1.0f : __builtin_amdgcn_exp2f(top - to);
      top = to;
      total *= by;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        acc[b] *= by;
    }
    const float less = top == -kInf ? 0.0f : top;
    float p[4 * kSets];
#pragma unroll
    for (int i = 0; i < 4 * kSets; ++i) {
      p[i] = __builtin_amdgcn_exp2f(fmaf(score[i / 4][i % 4], scale, -less));
      if constexpr (decltype(careful)::value)
        p[i] *= lower;
    }
    v2u weight[kSets][kWeightParts<T>];
#pragma unroll
    for (int s = 0; s < kSets; ++s)
      weight_parts(p + 4 * s, weight[s]);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float by = fp4_scale(x.value_scale[b]);
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        lds_write((along ^ (w << 4)) + 16 * b * Tile::kPitch,
                  fp4_values(x.value[b][w], by));
    }
    // Reads of two pairs of blocks across the values' rows are on their way before
    // the products, then one for each pair that is multiplied (the compiler, left
    // to itself, waits for every read).
    constexpr int kPairs = kBlocks / 2, kAhead = 2 < kPairs ? 2 : kPairs;
    v4u vf[kBlocks];
    auto read = [&](int pair) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 2 * pair; b < 2 * pair + 2; ++b) {
        const v2u lo = lds_read_across(across ^ (b << 5), 0);
        const v2u hi = lds_read_across(across ^ (b << 5), 16 * Tile::kPitch);
        vf[b] = v4u{lo.x, lo.y, hi.x, hi.y};
      }
    };
#pragma unroll
    for (int pair = 0; pair < kAhead; ++pair)
      read(pair);
    __builtin_amdgcn_sched_barrier(0);
    v4u by[kWeightParts<T>];
#pragma unroll
    for (int i = 0; i < kWeightParts<T>; ++i) {
      v2u run[2] = {weight[0][i], weight[kSets - 1][i]};
      if constexpr (kHalves) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          run[0][e] = row_of < ROWS ? run[0][e] : 0u;
          run[1][e] = row_of < ROWS ? 0u : run[1][e];
        }
      }
      by[i] = v4u{run[0].x, run[0].y, run[1].x, run[1].y};
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int pair = 0; pair < kPairs; ++pair) {
#pragma unroll
      for (int i = 0; i < kWeightParts<T>; ++i)
#pragma unroll
        for (int b = 2 * pair; b < 2 * pair + 2; ++b) {
          if constexpr (kApart) {
            const v4f first = mma16(v4u{vf[b].x, vf[b].y, 0, 0}, by[i], acc[b]);
            const v4f second = mma16(v4u{0, 0, vf[b].z, vf[b].w}, by[i], acc[b]);
            acc[b] = row_of < ROWS ? first : second;
          } else {
            acc[b] = mma16(vf[b], by[i], acc[b]);
          }
        }
#pragma unroll
      for (int i = pair; i < kWeightParts<T>; i += kPairs)
        total = mma16(ones, by[i], total);
      if (pair + kAhead < kPairs)
        read(pair + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  for (;;) {
    const int all = see.tiles();
    t0 = my.from - my.offset;
    const int end = args.shares == 0 ? all : my.to - my.offset; // the share's
    t1 = end > all ? all : end;
    static_assert(kSteps <= kThreads / kWave, ""); // (a step of queries a wave)
    if (wave < kSteps) {
      const int c = D / 4 * g + 8 * wave;
      const T *p = static_cast<const T *>(a.query) + seq * a.query_token +
                   (hk * a.group + first_row + row_of % ROWS) * a.query_head + c;
      Frag<T> x = live && c < a.d && !none ? ld_frag(p) : zero_frag<T>();
      if (a.alpha < 0.0f)
        x = negate_frag<T>(x);
      v4u cut[kQueryParts<T>];
      query_parts(x, cut);
#pragma unroll
      for (int i = 0; i < kQueryParts<T>; ++i)
        queries[(i * kSteps + wave) * kWave + lane] = cut[i];
    }
    __syncthreads();
    lower = 1.0f;
    bool some; // whether a key was there (wave-uniform)
    const int mine = t1 - t0 > wave ? (t1 - t0 - wave + 3) / 4 : 0;
    auto pass = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
        acc[b] = v4f{};
      total = v4f{};
      top = -kInf;
      some = false;
      for (int done = 0; done < mine; done += kWave / 2) {
        const int first = t0 + wave + 4 * done;
        const int n = mine - done < kWave / 2 ? mine - done : kWave / 2;
        const Runs runs = locate(first);
        Data x, y;
        fetch(x, runs, 0, see.first_key(first));
        if constexpr (kHalves && decltype(careful)::value) {
          // (the next tile's loads under way would need registers that the
          // products of single runs take)
          for (int k = 0;;) {
            some |= (x.has[0] | x.has[1]) != 0;
            compute(x, careful);
            if (++k == n)
              break;
            fetch(x, runs, k, see.first_key(first + 4 * k));
          }
          continue;
        }
        for (int k = 0; k < n; k += 2) {
          go_first(extent, end - (first + 4 * k));
          if (k + 1 < n)
            fetch(y, runs, k + 1, see.first_key(first + 4 * k + 4));
          some |= (x.has[0] | x.has[1]) != 0;
          compute(x, careful);
          if (k + 1 < n) {
            if (k + 2 < n)
              fetch(x, runs, k + 2, see.first_key(first + 4 * k + 8));
            some |= (y.has[0] | y.has[1]) != 0;
            compute(y, careful);
          }
        }
      }
    };
    pass(std::false_type{});
    // (a sum past fp32's range of values whose mean lies within: such columns
    // once more under lower probabilities, as in the attention of bf16 caches; or
    // a value that is infinite)
    const bool past = live && !all_finite(acc);
    if (ballot(past) != 0) {
      if (rows16_max(past ? 1.0f : 0.0f) != 0.0f)
        lower = __builtin_amdgcn_exp2f(-kLag - raise_of((t1 - t0) * kTile));
      pass(std::true_type{});
    }
    const float raise =
        lower == 1.0f ? 0.0f : kLag + raise_of((t1 - t0) * kTile);
    if (some && top == -kInf)
      top = kLowest;
    // (a share's first part may go on from the one before: slot 0)
    const int64_t of =
        (((int64_t)unit * args.shares + number) * 2 + (begun ? 1 : 0)) * ROWS;
    store_part<T, D, F::kWaveBytes, ROWS>(
        a, lds, found, top, total[0], raise, acc, rows, t0 == 0 && t1 == all,
        seq, hk, first_row, a.sums + of * D, a.stats + of * 2);
    begun = true;
    my.offset += all;
    my.from = my.offset;
    if (args.shares == 0 || my.from >= my.to)
      return;
    do {
      if (++seq >= a.sequences) // (only if lengths change under the call)
        return;
      see = uniform_tiles(a, seq);
    } while (see.count == 0);
    __syncthreads(); // (LDS of the part before is free)
  }
}

// The parts of a sequence's tiles in the shares of a unit: the first of these,
// how many, and their slot in the first one.
struct Parts {
  int first, count, slot;
};
template <int HELD>
__device__ __forceinline__ Parts parts_of(const Fp4StepArgs &args, int seq) {
  const int own = tiles_of(args.s, seq);
  const AllTiles<HELD> all(args.s);
  auto tiles = [](int n) { return n; };
  const int total = __builtin_amdgcn_readlane(sum_to_lane(all.sum(tiles)),
                                              kWave - 1);
  const Split split(args, total, all);
  // the sum over the sequences before this one
  const int lane = seq / all.each, within = seq - lane * all.each;
  auto before = [&](auto value) __attribute__((always_inline)) {
    const int sum = all.sum(value);
    return __builtin_amdgcn_readlane(
        sum_to_lane(sum) - sum + all.sum(within, value), lane);
  };
  Parts p{0, 0, 0};
  if (own == 0)
    return p;
  if (split.whole) {
    auto shares = [&](int n) { return split.shares(n); };
    p.first = before(shares);
    p.count = shares(own);
  } else {
    const int n = before(tiles);
    p.first = n / split.most;
    p.count = (n + own - 1) / split.most - p.first + 1;
    p.slot = n != p.first * split.most ? 1 : 0;
  }
  // (more only if lengths change under the call)
  const int left = args.shares - p.first;
  if (p.count > left)
    p.count = left > 0 ? left : 0;
  return p;
}

// Parts of a query head, joined: DIM / 32 consecutive elements a lane.
template <int N> struct Joined {
  float top = -kInf, l = 0.0f, o[N] = {};
  __device__ __forceinline__ void scale(float to) {
    const float by = top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to);
    top = to;
    l *= by;
#pragma unroll
    for (int e = 0; e < N; ++e)
      o[e] *= by;
  }
  // AT_ONCE of `count` parts, `step` apart: their loads are on their way together.
  template <int AT_ONCE, typename F>
  __device__ __forceinline__ void add(int from, int step, int count, float lower,
                                      F row) {
    typedef float Sums __attribute__((ext_vector_type(N)));
    const int c = lane_id() % 32 * N;
    Sums sums[AT_ONCE];
    float m[AT_ONCE], weight[AT_ONCE], to = top;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int part = from + i * step;
      const PartRow r = row(part < count ? part : 0);
      sums[i] = *reinterpret_cast<const Sums *>(r.sums + c);
      m[i] = r.stats[0];
      weight[i] = r.stats[1];
      if (part >= count) {
        sums[i] = Sums{};
        m[i] = -kInf;
        weight[i] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
      to = fmaxf(to, m[i]);
    scale(to);
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      weight[i] *= lower * (m[i] == to ? 1.0f
                                       : __builtin_amdgcn_exp2f(m[i] - to));
      l += weight[i];
#pragma unroll
      for (int e = 0; e < N; ++e)
        o[e] = fmaf(sums[i][e], weight[i], o[e]);
    }
  }
};

// The parts of the query heads of a sequence whose tiles several shares hold; zeros
// for one without a key.  THREADS / 256 is 1, a head a wave; or 4, one head, whose
// parts the half waves take in turn.
template <typename T, int DIM, int THREADS>
__global__ __launch_bounds__(THREADS) void fp4_cache_join(Fp4StepArgs args) {
  constexpr int N = DIM / 32, kHalves = THREADS / 32;
  constexpr int kHeads = THREADS == kThreads ? THREADS / kWave : 1;
  const StepArgs &a = args.s;
  const int of = (a.query_heads + kHeads - 1) / kHeads; // a sequence's workgroups
  const int seq = (int)(blockIdx.x / of);
  const int head = (int)(blockIdx.x - seq * of) * kHeads +
                   (kHeads > 1 ? wave_in_group() : 0);
  __shared__ Parts found; // (by one wave for all)
  if (wave_in_group() == 0) {
    const Parts p = a.sequences <= kWave ? parts_of<1>(args, seq)
                                         : parts_of<4>(args, seq);
    if (lane_id() == 0)
      found = p;
  }
  __syncthreads();
  const Parts parts{__builtin_amdgcn_readfirstlane(found.first),
                    __builtin_amdgcn_readfirstlane(found.count),
                    __builtin_amdgcn_readfirstlane(found.slot)};
  if (parts.count == 1 || head >= a.query_heads)
    return; // (it is written)
  const int hk = head / a.group, in_group = head - hk * a.group;
  const int block = in_group / args.block;
  const int64_t unit = hk * ((a.group + args.block - 1) / args.block) + block;
  const int64_t first =
      (unit * args.shares + parts.first) * 2 * args.block +
      (in_group - block * args.block);
  auto row = [&](int i) __attribute__((always_inline)) {
    const int64_t r = first + (2 * i + (i == 0 ? parts.slot : 0)) * args.block;
    return PartRow{a.sums + r * DIM, a.stats + r * 2};
  };
  T *out = static_cast<T *>(a.output) + seq * a.output_token +
           head * a.output_head;
  const int half = (int)threadIdx.x % (kHeads > 1 ? kWave : THREADS) / 32;
  constexpr int kStep = kHalves / kHeads;
  Joined<N> x;
  int from = half;
  if constexpr (kHeads > 1) // (8 at once for many parts in a wave)
    for (; from + 4 * kStep < parts.count; from += 8 * kStep)
      x.template add<8>(from, kStep, parts.count, a.lower, row);
  for (; from < parts.count; from += 4 * kStep)
    x.template add<4>(from, kStep, parts.count, a.lower, row);
  // both halves of a wave
  x.scale(fmaxf(x.top, shfl_xor32(x.top)));
  x.l += shfl_xor32(x.l);
#pragma unroll
  for (int e = 0; e < N; ++e)
    x.o[e] += shfl_xor32(x.o[e]);
  const int c = lane_id() % 32 * N;
  if constexpr (kHeads > 1) {
    if (lane_id() < 32 && c < a.d) {
      const float by = 1.0f / x.l;
#pragma unroll
      for (int e = 0; e < N; ++e)
        stv(out + c + e, x.top == -kInf ? 0.0f : x.o[e] * by);
    }
  } else {
    constexpr int kWaves = THREADS / kWave;
    __shared__ float outs[kWaves][DIM], tops[kWaves], totals[kWaves];
    const int wave = wave_in_group();
    if (lane_id() < 32) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        outs[wave][c + e] = x.o[e];
      tops[wave] = x.top;
      totals[wave] = x.l;
    }
    __syncthreads();
    if ((int)threadIdx.x >= a.d)
      return;
    float top = tops[0], l = 0.0f, o = 0.0f;
#pragma unroll
    for (int i = 1; i < kWaves; ++i)
      top = fmaxf(top, tops[i]);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float by =
          tops[i] == top ? 1.0f : __builtin_amdgcn_exp2f(tops[i] - top);
      l = fmaf(totals[i], by, l);
      o = fmaf(outs[i][threadIdx.x], by, o);
    }
    stv(out + threadIdx.x, top == -kInf ? 0.0f : o * (1.0f / l));
  }
}

// ---- host ------------------------------------------------------------------------

struct Plan {
  int64_t block, units, shares, sums, stats; // sums, stats: floats
  int64_t bytes() const { return 4 * (sums + stats); }
};

// Compute units, and the fewest tiles that a workgroup is made for (bf16, 32 heads
// over 8 of 128, us with 4, 8 and 16: one sequence of 1,024 keys 10.6, 11.5 and
// 13.5, eight of up to 1,024 12.9, 12.3 and 14.6, one of 32,768 19.8, 19.7 and
// 19.1, eight of up to 8,192 19.7, 19.7 and 18.2).
constexpr int64_t kUnits = 256, kLeast = 8;

// `waves`: workgroups of a compute unit.  Not split, a workgroup for each sequence
// and no join, are sequences of few keys, of not many where there are half as many
// of them as shares, and more of them than a share can be found among.  (us of
// sequences of up to so many keys, 32 heads over 8 of 128, bf16, split and not: 1 of
// 1,024 11.5 and 13.1, 8 of 1,024 12.3 and 14.7, 8 of 544 11.3 and 10.6, 32 of 2,048
// 21.8 and 25.4, 64 of 1,024 22 and 18.7, 64 of 2,048 33 and 30.6, 256 of 2,048 89
// and 84, 256 of 4,096 145.5 and 146.6; fp32: 64 of 1,024 26 and 23, 64 of 2,048
// 38.3 and 37.2, 256 of 4,096 170 and 172.  400 of 2,048, 16 heads over one: 38.5 and
// 31.)  Either way such batches are far from their bytes' time: 32 of 2,048 6.7, 64 of
// 1,024 6.5, of 2,048 14, 256 of 1,024 28 (50 here), of 2,048 55.
Plan plan(int64_t sequences, int64_t capacity, int64_t query_heads,
          int64_t key_heads, int64_t d, int64_t window, int64_t sinks,
          int64_t waves) {
  Plan p{};
  const int64_t group = query_heads / key_heads;
  p.block = group <= 8 ? 8 : kRows;
  p.units = key_heads * sw::ceil_div(group, p.block);
  const int64_t visible = most_visible(capacity, window, sinks);
  const int64_t shares = std::max<int64_t>(1, kUnits * waves / p.units);
  // (kWhole is _FP4_WHOLE of ../__init__.py)
  constexpr int64_t kWhole = 512;
  const int64_t few = std::min<int64_t>(2048, 4096 * sequences / shares);
  if (visible <= std::max(kWhole, few) || sequences > 4096 ||
      sequences * sw::ceil_div(capacity, 32) > sw::kMostTokens)
    return p;
  p.shares = shares;
  const int64_t all = p.units * p.shares * 2 * p.block;
  p.sums = all * (d <= 32 ? 32 : d <= 64 ? 64 : 128);
  p.stats = all * 2;
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
                      key_heads, d, window, sinks,
                      d <= 32   ? Fp4Parts<T, 32>::kWaves
                      : d <= 64 ? Fp4Parts<T, 64>::kWaves
                                : Fp4Parts<T, 128>::kWaves);
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
  a.window = (int)std::min<int64_t>(window, sw::kMostTokens);
  a.sinks = (int)std::min<int64_t>(sinks, sw::kMostTokens);
  a.alpha = alpha;
  args.block = (int)p.block;
  args.units = (int)p.units;
  args.shares = (int)p.shares;
  args.least = (int)kLeast;
  if (p.shares == 0)
    args.least = (int)sw::ceil_div(
        most_visible(page_size * table_width, window, sinks), kTile);
  a.lower = std::ldexp(
      1.0f, -(int)std::ceil(std::log2((double)(page_size * table_width + 64))) -
                1 - (int)kLag);
  a.sums = static_cast<float *>(workspace);
  a.stats = a.sums + p.sums;
  const int64_t grid = p.units * (p.shares ? p.shares : sequences);
  // Few rows take a workgroup of 1024 each (4 sequences of up to 100,000 keys, 12
  // heads over 4 of 128, bf16: 32.5 us of both kernels, 37.3 with a wave each; up to
  // 25,000 18.9 and 23.5); one of four rows else (256 sequences, 32 heads: the join
  // 19.8 us with one of 256 for each row).
  const bool few = sequences * query_heads <= 512;
  const int64_t join =
      sequences * (few ? query_heads
                       : sw::ceil_div(query_heads, kThreads / kWave));
  if (int rc = sw::check_flat_grid(std::max(grid, join), kThreads, what))
    return rc;
  const hipStream_t st = sw::as_stream(stream);
  const dim3 g((unsigned)grid);
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (a.group <= 8)
      fp4_cache_parts<T, D, 8, true><<<g, kThreads, 0, st>>>(args);
    else if (a.group <= kRows)
      fp4_cache_parts<T, D, kRows, true><<<g, kThreads, 0, st>>>(args);
    else
      fp4_cache_parts<T, D, kRows, false><<<g, kThreads, 0, st>>>(args);
  };
  if (d <= 32)
    launch(std::integral_constant<int, 32>{});
  else if (d <= 64)
    launch(std::integral_constant<int, 64>{});
  else
    launch(std::integral_constant<int, 128>{});
  if (int rc = sw::launch_check(what))
    return rc;
  if (p.shares == 0)
    return SW_OK;
  const dim3 j((unsigned)join);
  auto launch_join = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (few)
      fp4_cache_join<T, D, 4 * kThreads><<<j, 4 * kThreads, 0, st>>>(args);
    else
      fp4_cache_join<T, D, kThreads><<<j, kThreads, 0, st>>>(args);
  };
  if (d <= 32)
    launch_join(std::integral_constant<int, 32>{});
  else if (d <= 64)
    launch_join(std::integral_constant<int, 64>{});
  else
    launch_join(std::integral_constant<int, 128>{});
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
              window, sinks, d <= 32 ? 5 : 4).bytes(); // (the most of any type)
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
