// Device-side building blocks of attention over [tokens][heads][d] operands:
// fragments of the matrix cores, tiles of rows in LDS that are read both
// along and across their rows, and the search for a packed sequence.
//
// A matrix product of 32 x 32 with K = 16 takes from lane l the eight
// elements k = 8 (l / 32) + i of row (A) or column (B) l % 32, and leaves in
// accumulator r of lane l the element of row 8 (r / 4) + 4 (l / 32) + r % 4
// and column l % 32.  The eight accumulators 8 s .. 8 s + 7 of a result are
// therefore a B operand of the next product as they stand, for the K indices
// 16 s + 8 (i / 4) + 4 (l / 32) + i % 4: scores are computed as K Q^T, keys
// in rows and queries in columns, and the probabilities stay in registers.
// The A operand of that product runs across the rows of a tile (V^T, or K^T
// in a gradient): bf16 tiles are read by the transposing LDS load, which
// gives lane i of 16 column i of four rows.
#pragma once

#include "sw_device.h"

namespace swd {

typedef float v8f __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

template <typename T> struct FragOf;
template <> struct FragOf<float> { using type = v8f; };
template <> struct FragOf<uint16_t> { using type = v4u; };
template <typename T> using Frag = typename FragOf<T>::type;

__device__ __forceinline__ v16f mma32(v4u a, v4u b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
      0);
}
// fp32 has K = 2 a product, one index of each half of the wave: element i of
// both halves is product i, so the fragments are those of bf16
__device__ __forceinline__ v16f mma32(v8f a, v8f b, v16f c) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ v4f mma16(v4u a, v4u b, v4f c) {
  return mfma_16x16x32_bf16(a, b, c);
}
__device__ __forceinline__ v4f mma16(v8f a, v8f b, v4f c) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// Two fp32 values as bf16 in one instruction, the first in the low half.
__device__ __forceinline__ uint32_t cvt_pk_bf16(float lo, float hi) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t,
                            __builtin_convertvector(v2f{lo, hi}, bf16x2));
}

// Eight fp32 values as a fragment (bf16: each rounded to nearest even).
template <typename T> __device__ __forceinline__ Frag<T> make_frag(const float *x) {
  if constexpr (sizeof(T) == 4)
    return v8f{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
  else
    return v4u{cvt_pk_bf16(x[0], x[1]), cvt_pk_bf16(x[2], x[3]),
               cvt_pk_bf16(x[4], x[5]), cvt_pk_bf16(x[6], x[7])};
}
// Eight fp32 values that are not negative as the sum of two bf16 fragments, to
// 2^-15 of each: what their upper halves hold, and the rest of it, rounded.  The
// rest of a value that is not zero is at least 2^-126, so that an infinity times
// both parts is infinite twice, not NaN where nothing is left.
__device__ __forceinline__ void split_frag(const float *x, v4u &upper,
                                           v4u &rest) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    r[e] = __builtin_amdgcn_fmed3f(
        x[e] - __uint_as_float(__float_as_uint(x[e]) & 0xFFFF0000u), 0x1p-126f,
        x[e]);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    upper[e] = __builtin_amdgcn_perm(__float_as_uint(x[2 * e + 1]),
                                     __float_as_uint(x[2 * e]), 0x07060302u);
  rest = make_frag<uint16_t>(r);
}
template <typename T> __device__ __forceinline__ Frag<T> zero_frag() {
  if constexpr (sizeof(T) == 4)
    return v8f{0, 0, 0, 0, 0, 0, 0, 0};
  else
    return v4u{0, 0, 0, 0};
}
// The fragment with element i alone, in the lanes where `keep` holds.
template <typename T>
__device__ __forceinline__ Frag<T> one_of_frag(Frag<T> f, int i, bool keep) {
  Frag<T> r = zero_frag<T>();
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      r[e] = keep && e == i ? f[e] : 0.0f;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r[e] = keep && e == i / 2 ? f[e] & (i % 2 ? 0xFFFF0000u : 0xFFFFu) : 0u;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ Frag<T> negate_frag(Frag<T> f) {
  if constexpr (sizeof(T) == 4)
    return -f;
  else
    return f ^ 0x80008000u;
}
// sum of the products of two fragments' elements
template <typename T>
__device__ __forceinline__ float dot_frag(Frag<T> a, Frag<T> b, float c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      c = fmaf(a[e], b[e], c);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c = fmaf(bf16_to_f32(a[e] & 0xFFFFu), bf16_to_f32(b[e] & 0xFFFFu), c);
      c = fmaf(__uint_as_float(a[e] & 0xFFFF0000u),
               __uint_as_float(b[e] & 0xFFFF0000u), c);
    }
  }
  return c;
}

// Eight elements from 16-byte aligned global memory.
__device__ __forceinline__ v4u ld_frag(const uint16_t *p) {
  return *reinterpret_cast<const v4u *>(p);
}
__device__ __forceinline__ v8f ld_frag(const float *p) {
  const v4f a = *reinterpret_cast<const v4f *>(p);
  const v4f b = *reinterpret_cast<const v4f *>(p + 4);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Four consecutive fp32 values to an 8 (bf16) or 16 (fp32) byte aligned place.
__device__ __forceinline__ void st4(float *p, float a, float b, float c,
                                    float d) {
  *reinterpret_cast<v4f *>(p) = v4f{a, b, c, d};
}
__device__ __forceinline__ void st4(uint16_t *p, float a, float b, float c,
                                    float d) {
  *reinterpret_cast<v2u *>(p) = v2u{cvt_pk_bf16(a, b), cvt_pk_bf16(c, d)};
}

// The value of lane l ^ 32 combined with the lane's own, in both.
__device__ __forceinline__ float both_halves_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(
      __float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float both_halves_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(
      __float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// ---- results that are not finite -----------------------------------------------
// Whether a lane's accumulators all are (V: a vector of fp32).
template <typename V, int BLOCKS>
__device__ __forceinline__ bool all_finite(const V (&acc)[BLOCKS]) {
  float x = 0.0f;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int r = 0; r < (int)(sizeof(V) / 4); ++r)
      x = fmaf(acc[b][r], 0.0f, x);
  return x == 0.0f;
}
// Whether a wave of the workgroup says so; every thread must call it.
__device__ __forceinline__ bool any_wave(bool says, int *verdict) {
  if (threadIdx.x == 0)
    *verdict = 0;
  __syncthreads();
  if (ballot(says) != 0 && lane_id() == 0)
    *verdict = 1;
  __syncthreads();
  return *verdict != 0;
}
// For a sum of up to n values (n < 2^31) under weights of at most 1, each
// rounded: the power of two by which the weights are lowered so that no sum of
// them passes the largest value.
__device__ __forceinline__ float raise_of(int n) {
  return (float)(33 - __builtin_clz(n | 1));
}

// ---- LDS by address ----------------------------------------------------------
// Addresses are byte offsets in the workgroup's LDS: a lane's part and a part
// known when the kernel is built, which becomes the instruction's offset.
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t lane, uint32_t at) {
  return *(const __attribute__((address_space(3))) V *)(uintptr_t)(lane + at);
}
template <typename V>
__device__ __forceinline__ void lds_write(uint32_t at, V v) {
  *(__attribute__((address_space(3))) V *)(uintptr_t)at = v;
}
// the transposing load of 16-bit elements: lane i of 16 reads 8 bytes, and gets
// the elements i % 4 of what lanes i / 4, i / 4 + 4, + 8, + 12 of its 16 read
__device__ __forceinline__ v2u lds_read_across(uint32_t lane, uint32_t at) {
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                     (lds_v4s *)(uintptr_t)(lane + at)));
}

// The words of buffer_rsrc(p, n), for an instruction written out.
__device__ __forceinline__ v4u buffer_words(const void *p, uint32_t n) {
  const uint64_t a = (uint64_t)p;
  return v4u{(uint32_t)__builtin_amdgcn_readfirstlane((int)a),
             (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) & 0xFFFFu,
             (uint32_t)__builtin_amdgcn_readfirstlane((int)n), 0x00020000u};
}
// Starts a copy of 16 bytes a lane from the buffer to 1024 consecutive bytes
// of LDS at the wave-uniform address.  Written out because the compiler waits
// for every copy that its builtin has under way before the next LDS read, of
// whichever tile (which made each tile wait for the next one's copy); this one
// returns no register, and landed() waits for it.  It sets m0, which the
// compiler keeps for itself and sets before instructions that read it: the
// clobber keeps such a value from being carried across, and the warning that
// this draws (m0 is not preserved) says what is meant.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(v4u buffer, uint32_t at,
                                            uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\t"
               "buffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(at),
                 "s"(buffer)
               : "memory", "m0");
}

// The same of 4 bytes a lane, to 256 consecutive bytes.
__device__ __forceinline__ void copy_words_to_lds(v4u buffer, uint32_t at,
                                                  uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\t"
               "buffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(at),
                 "s"(buffer)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// For N products of this stretch of code, each with one LDS read of its own:
// four reads first, then a product and a read in turn, so that a product waits
// for a read of four before it.  (The compiler otherwise leaves two reads in
// flight.)
template <int N> __device__ __forceinline__ void schedule_reads() {
  constexpr int kProduct = 0x8, kRead = 0x100, kAhead = 4;
  if constexpr (N > kAhead) {
    __builtin_amdgcn_sched_group_barrier(kRead, kAhead, 0);
#pragma unroll
    for (int i = 0; i < N - kAhead; ++i) {
      __builtin_amdgcn_sched_group_barrier(kProduct, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kProduct, kAhead, 0);
  }
}

// ---- tiles of rows in LDS ----------------------------------------------------
// Rows of D elements without padding, in chunks of 16 bytes; chunk c of row r
// lies at place c ^ swizzle(r).  The swizzle keeps these reads free of bank
// conflicts (64 banks of 4 bytes): 16 consecutive rows at one chunk (a
// fragment along the rows), and, for bf16, four consecutive chunks of each of
// four consecutive rows or two of each of eight (half a wave's transposing
// load for products of 32 or 16 rows).  ROWS is a multiple of 32 and a tile is
// filled by THREADS threads.
template <typename T, int D, int ROWS, int THREADS> struct RowTile {
  static constexpr int kChunks = D * (int)sizeof(T) / 16;
  static constexpr int kPitch = D * (int)sizeof(T);
  static constexpr int kBytes = ROWS * kPitch;
  static constexpr int kPasses = ROWS * kChunks / THREADS;
  static constexpr int kSteps = D / 16; // products along a row
  static_assert(ROWS * kChunks % THREADS == 0 && 1024 % kPitch == 0, "");

  __device__ static __forceinline__ int swizzle(int row) {
    if constexpr (sizeof(T) == 4)
      return row & 15;
    else if constexpr (kChunks == 16)
      return ((row & 3) << 2) | ((row >> 1) & 2) | ((row >> 3) & 1);
    else
      return ((row << 1) & 4) | ((row >> 1) & 2) | ((row >> 3) & 1);
  }
  __device__ static __forceinline__ int place(int row, int chunk) {
    return row * kPitch + ((chunk ^ swizzle(row)) << 4);
  }

  // Starts the copy of rows 0 .. rows - 1 of the matrix at `base`
  // (wave-uniform; row_bytes apart, d elements of each) to the tile at `lds`,
  // without registers between: a wave's load writes 1024 consecutive bytes of
  // LDS, and each lane picks the chunk that belongs at its place.  Elements
  // past d and rows past the end are written as zeros (the descriptor bounds
  // what is read: (ROWS - 1) row_bytes + 4 D < 2^31 is the host's check).
  // landed() waits for it.  `w`: this wave's number among the THREADS / 64 that
  // fill the tile.
  __device__ static __forceinline__ void copy(uint32_t lds, const T *base,
                                              int rows, uint32_t row_bytes,
                                              int d, int w) {
    const int l = lane_id();
    constexpr int kStep = (THREADS / kWave) * (1024 / kPitch); // rows a pass
    rows = rows < 0 ? 0 : rows > ROWS ? ROWS : rows;
    const uint32_t bytes =
        rows == 0 ? 0u : (uint32_t)(rows - 1) * row_bytes + d * sizeof(T);
    const v4u buffer = buffer_words(base, bytes);
    uint32_t at = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int row = w * (1024 / kPitch) + l / kChunks;
      if (p == 0 || kStep % 16 != 0) { // (the swizzle has a period of 16 rows)
        const int c = (l % kChunks) ^ swizzle(row + p * kStep);
        // (an offset past every descriptor: reads zero)
        at = c * 16 < d * (int)sizeof(T) ? row * row_bytes + c * 16
                                         : 0x80000000u;
      }
      copy_to_lds(buffer, at + p * kStep * row_bytes,
                  lds + (p * (THREADS / kWave) + w) * 1024);
    }
  }

  // A lane's addresses within any tile, in two registers: an operation for each
  // address that is used.
  struct FewLane {
    uint32_t x, y;
    __device__ __forceinline__ FewLane() {
      const int l = lane_id(), h = l >> 5, i = l & 15;
      if constexpr (sizeof(T) == 2) {
        x = place(l & 31, h);
        y = place(4 * h + (i >> 2), 2 * ((l >> 4) & 1) + ((i & 3) >> 1)) +
            (i & 1) * 8;
      } else {
        x = place(l & 31, 2 * h);
        y = place(4 * h, (l & 31) >> 2) + (l & 3) * 4;
      }
    }
    // (a multiple of 512: the operations below change bits under it)
    __device__ __forceinline__ void offset(uint32_t by) {
      x += by;
      y += by;
    }
    // (keeps the compiler from computing every address ahead of a loop)
    __device__ __forceinline__ void fresh() {
      asm volatile("" : "+v"(x), "+v"(y));
    }
    // bf16: chunk 2 i + h; fp32: chunk 4 (i / 2) + 2 h + i % 2
    __device__ __forceinline__ uint32_t along(int i) const {
      return x ^ (sizeof(T) == 2 ? i << 5 : (i >> 1) << 6 | (i & 1) << 4);
    }
    // bf16: chunks from 4 (i % (D / 32)) on, rows from 8 (i / (D / 32)) on;
    // fp32: row i
    __device__ __forceinline__ uint32_t across(int i) const {
      if constexpr (sizeof(T) == 2)
        return (y ^ ((i % (D / 32)) << 6 | (i / (D / 32)) << 4)) +
               i / (D / 32) * 8 * kPitch;
      else
        return (y ^ (i << 4)) + i * kPitch;
    }
  };
  // The same computed once: what is left of a read's address is a constant that
  // the load instruction adds.
  // (The swizzle reaches the chunk's four low bits: fp32 reads that differ in
  // higher ones share an address.)
  struct Lane {
    uint32_t x[sizeof(T) == 2 ? kSteps : 8], y[sizeof(T) == 2 ? 2 * (D / 32) : 4];
    __device__ __forceinline__ Lane() {
      const FewLane f;
#pragma unroll
      for (int i = 0; i < (int)(sizeof x / 4); ++i)
        x[i] = f.along(i);
#pragma unroll
      for (int i = 0; i < (int)(sizeof y / 4); ++i)
        y[i] = f.across(i);
    }
    __device__ __forceinline__ void offset(uint32_t by) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof x / 4); ++i)
        x[i] += by;
#pragma unroll
      for (int i = 0; i < (int)(sizeof y / 4); ++i)
        y[i] += by;
    }
    __device__ __forceinline__ uint32_t along(int i) const { return x[i]; }
    __device__ __forceinline__ uint32_t across(int i) const { return y[i]; }
  };
  // Row 32 rb + l % 32, elements 16 s + 8 (l / 32) + i: the A operand with
  // the tile's rows as rows (or B, with its rows as columns).
  template <typename L>
  __device__ static __forceinline__ Frag<T> along(uint32_t lds, const L &n,
                                                  int rb, int s) {
    const uint32_t at = lds + 32 * rb * kPitch;
    if constexpr (sizeof(T) == 2) {
      return lds_read<v4u>(n.along(s), at);
    } else {
      const uint32_t up = at + 256 * (s / 4);
      const v4f a = lds_read<v4f>(n.along(2 * (s % 4)), up);
      const v4f b = lds_read<v4f>(n.along(2 * (s % 4) + 1), up);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // Element 32 db + l % 32 of the rows 16 st + 8 (i / 4) + 4 (l / 32) + i % 4:
  // the A operand with the tile's columns as rows, whose K indices are those
  // of accumulators 8 (st % 2) .. of row block st / 2.
  template <typename L>
  __device__ static __forceinline__ Frag<T> across(uint32_t lds, const L &n,
                                                   int st, int db) {
    const uint32_t at = lds + 16 * st * kPitch;
    if constexpr (sizeof(T) == 2) {
      const v2u x = lds_read_across(n.across(db), at);
      const v2u y = lds_read_across(n.across(D / 32 + db), at);
      return v4u{x.x, x.y, y.x, y.y};
    } else {
      v8f r;
#pragma unroll
      for (int i = 0; i < 8; ++i) // (row bit 3 swaps chunks 8 apart)
        r[i] = lds_read<float>(n.across(i & 3),
                               at + 8 * (i >> 2) * kPitch +
                                   128 * ((db ^ (i >> 2)) & 1) +
                                   256 * (db >> 1));
      return r;
    }
  }
};

// Waits until this wave's copies and its reads of earlier tiles are done.
__device__ __forceinline__ void landed_wave() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}
// Waits until this wave's copies and its reads of earlier tiles are done, and
// then for the workgroup's other waves.
__device__ __forceinline__ void landed() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A lane's row of 32 as fragments, zeros where it is not live and past d.
template <typename T, int STEPS>
__device__ __forceinline__ void load_rows(Frag<T> (&f)[STEPS], const T *p,
                                          bool live, int d, bool negate) {
  const int h = lane_id() >> 5;
#pragma unroll
  for (int st = 0; st < STEPS; ++st) {
    const int c = 16 * st + 8 * h;
    f[st] = live && c < d ? ld_frag(p + c) : zero_frag<T>();
    if (negate)
      f[st] = negate_frag<T>(f[st]);
  }
}

// ---- packed sequences ----------------------------------------------------------
// The last i of 0 .. n - 1 whose value(i) is at most x, 0 where none is; the
// values do not fall.  x is wave-uniform and so is the result; 64 probes a trip.
template <typename F>
__device__ __forceinline__ int last_at_most(int n, int x, F value) {
  const int l = lane_id();
  int from = 0, count = n; // the answer lies in [from, from + count)
  while (count > 1) {
    const int step = (count + kWave - 1) / kWave;
    const int at = from + l * step;
    const bool in = l * (int64_t)step < count;
    const int first = value(in ? at : from);
    // (probe 0 is at or before the answer: `from` starts there)
    const uint64_t before = ballot(in && first <= x);
    const int k = before ? 63 - __builtin_clzll(before) : 0;
    count = count - k * step < step ? count - k * step : step;
    from += k * step;
  }
  return __builtin_amdgcn_readfirstlane(from);
}

// Sequence i of n holds tokens offsets[i] .. offsets[i + 1] - 1, and, cut into
// tiles of 1 << shift tokens, the tile numbers (offsets[i] >> shift) + i up to
// that of i + 1: at least as many as it has tiles, without a count of the
// tiles before it.  Returns the sequence of tile number `tile`.
__device__ __forceinline__ int sequence_of_tile(
    const int32_t *__restrict__ offsets, int n, int tile, int shift) {
  return last_at_most(n, tile,
                      [&](int i) { return (offsets[i] >> shift) + i; });
}

} // namespace swd
