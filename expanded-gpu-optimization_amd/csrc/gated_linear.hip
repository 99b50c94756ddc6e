// Gated linear layer (fhoad_gated_linear_forward / _backward): h = act(x Wg^T + bg) * (x Wu^T + bu)
// and its gradients, as tiled matrix products on the bf16 matrix cores.
//
//   forward:  both projections of a tile in one kernel: a workgroup's columns are gate rows and up
//             rows of the same features, so g and u meet in one lane's accumulators and only h (and
//             for training g and u, in float32) is written.
//   backward: dg = dh u act'(g), du = dh act(g) side by side in [rows][2 padded hidden], then two
//             products, dx = [dg du] [Wg; Wu] and [dWg; dWu] = [dg du]^T x.
//
// float32 operands are split when a tile is staged, at float32 precision: into three bf16 parts and
// six products, or for the larger layers, after a pass that finds each row's scale, into two float16
// parts and three products (see the formats below): a sixth or a third of the bf16 rate, against a
// sixteenth with the float32 matrix instructions. bfloat16 operands are used as they are; dg and du
// are then rounded to bfloat16 once, as operands: the gradients' error is 0.0023 of their norm where the
// results' own rounding makes 0.0017, and in two parts each would double the products' time.
//
// 4 rows width hidden operations forward and twice that backward: but for the smallest batches
// the matrix cores bound it.
#include "network_common.h"

#include <algorithm>
#include <type_traits>

namespace fhoad_net {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

// ---- activations ------------------------------------------------------------------------------

// e^x to about an ulp, from the hardware's 2^y: the rounding of x log2(e) is put back as a first-order
// term, of either sign. Where 2^y is infinite (from y = 128, x = 88.7) the term would make it NaN, and an
// infinite x has none: from |y| = 128 on 2^y stays as it is, infinite or, below, zero.
__device__ __forceinline__ float exponential(float x) {
  const float y = x * 1.44269504f;
  float rest = __builtin_fmaf(x, 1.44269504f, -y);
  rest = __builtin_fmaf(x, 1.92596299e-8f, rest);  // log2(e) - its float32
  const float e = __builtin_amdgcn_exp2f(y);
  return __builtin_fabsf(y) < 128.0f ? __builtin_fmaf(e, rest * 0.693147181f, e) : e;
}

struct Activated {
  float value, slope;
};

// act(g) and act'(g). Written for few instructions: an epilogue has 128 of them to a lane, and
// library exp, tanh and erf (60 instructions and more) took a third of a product's time. The slopes
// come from e^-g and not from differences of rounded values, so they keep their relative precision
// where a unit saturates.
__device__ __forceinline__ Activated activate(int kind, float g) {
  switch (kind) {
    case FHOAD_TANH: {
      // tanh |g| = (1 - e) / (1 + e) with e = e^-2|g|; below 0.35 the series to g^11.
      const float magnitude = __builtin_fabsf(g);
      const float e = exponential(-2.0f * magnitude);
      const float q = __builtin_amdgcn_rcpf(1.0f + e);
      const float square = g * g;
      float series = __builtin_fmaf(square, -8.8632355e-3f, 2.1869489e-2f);
      series = __builtin_fmaf(square, series, -5.3968254e-2f);
      series = __builtin_fmaf(square, series, 0.133333333f);
      series = __builtin_fmaf(square, series, -0.333333333f);
      const float near_zero = __builtin_fmaf(magnitude * square, series, magnitude);
      const float value = magnitude < 0.35f ? near_zero : (1.0f - e) * q;
      return {__builtin_copysignf(value, g), 4.0f * e * q * q};
    }
    case FHOAD_GELU: {
      // Phi(-|g|) = e^(-g^2/2) Q(t), t = 1 / (1 + 0.33 |g|): Q is a least-maximum fit of
      // erfcx(|g| / sqrt 2) / 2 on 0 <= |g| <= 14 (1e-8 relative), where the exponential ends.
      const float magnitude = __builtin_fabsf(g);
      const float square = g * g;
      const float e = exponential(-0.5f * square);
      const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.33f, magnitude, 1.0f));
      float q = -0.026107169687747955f;
      q = __builtin_fmaf(q, t, 0.14980316162109375f);
      q = __builtin_fmaf(q, t, -0.3250703513622284f);
      q = __builtin_fmaf(q, t, 0.295117050409317f);
      q = __builtin_fmaf(q, t, -0.10955014824867249f);
      q = __builtin_fmaf(q, t, 0.147301584482193f);
      q = __builtin_fmaf(q, t, 0.10326091945171356f);
      q = __builtin_fmaf(q, t, 0.13376924395561218f);
      q = __builtin_fmaf(q, t, 0.13146893680095673f);
      q = __builtin_fmaf(q, t, 6.783101980545325e-06f);
      const float tail = e * q;
      const float below = g < 0.0f ? tail : 1.0f - tail;
      return {g * below, __builtin_fmaf(g * e, 0.398942280f, below)};
    }
    default: {
      const float e = exponential(-g);
      const float s = __builtin_amdgcn_rcpf(1.0f + e);
      const float rest = __builtin_fminf(e, 3e38f) * s;  // 1 - s
      if (kind == FHOAD_SIGMOID) return {s, s * rest};
      return {g * s, s * __builtin_fmaf(g, rest, 1.0f)};
    }
  }
}

// ---- operands ---------------------------------------------------------------------------------

// Two values rounded to bf16, a in the low half.
__device__ __forceinline__ unsigned bf16_pair(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f2{a, b}), bf2));
}

// The three bf16 parts of two values, each rounded to nearest: x = hi + mid + lo exactly (for
// |x| from 1e-32 up; below, parts may be subnormal bf16 values, which the matrix cores take as zero: 2^-126
// of x at most). The 2^15 float32 values next to the largest, which would round to an infinite hi, take the
// largest bf16 instead, and their remainders are whole again (this selection takes 1 to 3 % of the time of
// layers of 256 to 6,000 rows). An infinite value has a NaN remainder: what is formed from it is NaN.
__device__ __forceinline__ void split_pair(float a, float b, unsigned& hi, unsigned& mid, unsigned& lo) {
#pragma clang fp contract(off)
  constexpr float kMost = 0x1.FEp127f;
  hi = bf16_pair(__builtin_amdgcn_fmed3f(a, -kMost, kMost), __builtin_amdgcn_fmed3f(b, -kMost, kMost));
  a -= __builtin_bit_cast(float, hi << 16);
  b -= __builtin_bit_cast(float, hi & 0xffff0000u);
  mid = bf16_pair(a, b);
  a -= __builtin_bit_cast(float, mid << 16);
  b -= __builtin_bit_cast(float, mid & 0xffff0000u);
  lo = bf16_pair(a, b);
}

// Two float16 parts of two values that are scaled to below 2^15: x = hi + 2^-11 lo. lo, the scaled
// remainder, is about as large as hi, so both stay clear of float16's smallest values for 29 powers of
// two: the sum is x to 2^-23 of it down to 2^-14, and to 2^-36 (a 2^51st of the largest) below. The
// matrix cores take subnormal float16 values as they are.
__device__ __forceinline__ void split_half_pair(float a, float b, unsigned& hi, unsigned& lo) {
#pragma clang fp contract(off)
  typedef _Float16 half2 __attribute__((ext_vector_type(2)));
  const half2 h = __builtin_convertvector((f2{a, b}), half2);
  const float ha = static_cast<float>(h[0]), hb = static_cast<float>(h[1]);
  const half2 l = __builtin_convertvector((f2{(a - ha) * 2048.0f, (b - hb) * 2048.0f}), half2);
  hi = __builtin_bit_cast(unsigned, h);
  lo = __builtin_bit_cast(unsigned, l);
}

// How values become matrix operands.
//   Bf16:      bfloat16 values as they are, one product.
//   Bf16Parts: float32 values as three bf16 parts, six products (the other three are below 2^-24 of
//              a product). No preparation, every magnitude: the smaller products take it.
//   HalfParts: float32 values as two float16 parts, three products, hi hi and the two with a lo in
//              accumulators of their own, 2^11 apart. The fourth, lo lo, is left out: at most 2^-22 of a
//              product, and that much and of one sign where both values are 1 + 2^-11 (above 2^-24 for 13 %
//              of uniformly drawn pairs). With the parts' own 2^-23 of each value a product is good to 2^-21,
//              and a sum to that of its products' magnitudes. Half the matrix instructions, which bound the large products, but float16's range needs each row
//              scaled by a power of two to its largest value (a pass over the operands first), and
//              twice the accumulators halve the tile (input gradient at 65,536 x 1,024 x 2,731: 300
//              TFLOP/s; with lo unscaled and one set of accumulators 366, but then what is a 2^18th of
//              its row's largest value begins to lose digits, here what is a 2^29th). Bf16Parts: 217.
struct Bf16 {
  typedef __bf16 T;
  static constexpr int kParts = 1, kProducts = 1;
  static constexpr bool kScaled = false;
  static __device__ __forceinline__ constexpr int part_a(int) { return 0; }
  static __device__ __forceinline__ constexpr int part_b(int) { return 0; }
};
struct Bf16Parts {
  typedef float T;
  static constexpr int kParts = 3, kProducts = 6;  // smallest first
  static constexpr bool kScaled = false;
  static __device__ __forceinline__ constexpr int part_a(int k) { return k == 0 ? 2 : k == 1 || k == 3 ? 1 : 0; }
  static __device__ __forceinline__ constexpr int part_b(int k) { return k == 2 ? 2 : k == 1 || k == 4 ? 1 : 0; }
};
struct HalfParts {
  typedef float T;
  static constexpr int kParts = 2, kProducts = 3;
  static constexpr bool kScaled = true;
  static __device__ __forceinline__ constexpr int part_a(int k) { return k == 0 ? 1 : 0; }
  static __device__ __forceinline__ constexpr int part_b(int k) { return k == 1 ? 1 : 0; }
};

// The power of two that brings a row's largest magnitude (its bits) to [2^14, 2^15); 0 for a row with a
// non-finite value, whose results are non-finite either way.
__device__ __forceinline__ int shift_of(unsigned top_bits) {
  const int exponent = static_cast<int>(top_bits >> 23);
  return exponent == 255 ? 0 : min(141 - exponent, 126);
}
__device__ __forceinline__ float power_of_two(int shift) {
  return __builtin_bit_cast(float, static_cast<unsigned>(127 + shift) << 23);
}

// Where a tile's rows and its depth (the contracted dimension) lie in memory:
//   kRows:          element (row, k) at base[row ld + k]
//   kPairedRows:    the same, rows alternating between two matrices (see paired_row)
//   kColumns:       element (row, k) at base[k ld + row]
//   kPairedColumns: the same, k up to `half` from the first matrix and beyond it from the second,
//                   of which the first `segment` of each half exist (zero between)
enum Source { kRows, kPairedRows, kColumns, kPairedColumns };

struct Matrix {
  const void* first;
  const void* second;
  int64_t ld;
  int64_t rows;     // rows that exist
  int64_t depth;    // k that exist (kPairedColumns: 2 half)
  int64_t half, segment;
  // HalfParts: the bits of each row's largest magnitude (kPairedRows: of both matrices').
  const unsigned* top;
  const unsigned* second_top;
  int64_t part;  // split operands (kPlanes): values from one part to the next
};

// Loads that need an element's alignment only (rows of odd length): the hardware takes any address.
template <typename V, typename T>
struct __attribute__((packed, aligned(alignof(T)))) Loose {
  V v;
};
template <typename V, typename T>
__device__ __forceinline__ V load_loose(const T* p) {
  return reinterpret_cast<const Loose<V, T>*>(p)->v;
}

// Geometry of a tile product: kM x kN results of a workgroup of kWavesM x kWavesN waves, kDepth
// deep at a time. Operand rows lie in LDS as chunks of 8 k (16 bytes), each part apart.
// kShortSums: a float32 tile forms each 16 k's six products apart and adds them to the results by
// themselves, a sixth of the roundings of one long sum (one row of 3,359: 1.8e-6 -> 0.8e-6 of the
// norm), for a tenth of the speed; the smallest products, which the matrix cores do not bound, take it.
template <typename Format_, int kM_, int kN_, int kWavesM_, int kWavesN_, int kDepth_, bool kShortSums_ = false>
struct Tile {
  typedef Format_ Format;
  typedef typename Format::T T;
  static constexpr bool kShortSums = kShortSums_;
  static constexpr int kM = kM_, kN = kN_, kDepth = kDepth_;
  static constexpr int kWavesM = kWavesM_, kWavesN = kWavesN_;
  static constexpr int kThreads = kWavesM * kWavesN * kWave;
  static constexpr int kParts = Format::kParts;
  static constexpr int kWaveM = kM / kWavesM, kWaveN = kN / kWavesN;
  static constexpr int kBlocksM = kWaveM / 32, kBlocksN = kWaveN / 32;
  static constexpr int kChunks = kDepth / 8;
  // 16-byte units of a row. Sixteen lanes that read one chunk of sixteen consecutive rows have to
  // meet sixteen different units modulo 16 (256 bytes of banks): an odd pitch does that, or, with
  // four or eight chunks, an exclusive or with the row over the rows that 256 bytes hold (with the
  // row itself, every second read conflicted).
  static constexpr bool kSwizzled = kChunks == 8 || kChunks == 4;
  static constexpr int kPitch = kSwizzled ? kChunks : kChunks + 1 - kChunks % 2;
  static __device__ __forceinline__ int swizzled(int row, int chunk) {
    return kSwizzled ? chunk ^ ((row / (16 / kChunks)) % kChunks) : chunk;
  }
};

// LDS row r of a paired tile: within a wave's columns, the first half are gate rows, the second up
// rows, of the same features.
template <typename G>
__device__ __forceinline__ int paired_feature(int r) {
  return (r / G::kWaveN) * (G::kWaveN / 2) + r % (G::kWaveN / 2);
}
template <typename G>
__device__ __forceinline__ bool paired_second(int r) {
  return r % G::kWaveN >= G::kWaveN / 2;
}

// Stages one operand of a tile (kOperandRows rows from `row0`, its LDS units from `lds0`): fetch()
// takes a depth step into registers, 8 values at a time as they lie in memory, stage() writes them
// to LDS as parts, operand() reads a lane's 8 k of one row back. Operands by rows lie in LDS by
// rows. Operands by columns lie there by columns of the tile, 8 rows to a 16-byte unit, and are
// transposed by the LDS read itself (ds_read_b64_tr_b16: 16 lanes read four k of 16 rows and each
// gets the four k of its row).
// Rows past the matrix's end repeat the last one or are zero (their results are not stored); depth
// past its end is zero.
template <typename G, Source kSource, int kOperandRows>
struct Stager {
  typedef typename G::T T;
  static constexpr bool kByColumns = kSource == kColumns || kSource == kPairedColumns;
  static constexpr int kPer = kOperandRows * G::kChunks / G::kThreads;  // 8-value chunks of a thread
  static_assert(kPer * G::kThreads == kOperandRows * G::kChunks, "whole chunks a thread");
  static constexpr int kAcross = kOperandRows / 8;  // by columns: units of one k
  static constexpr int kUnits = G::kParts * (kByColumns ? G::kDepth * kAcross : kOperandRows * G::kPitch);
  // The four k that 16 lanes read at once, 64 bytes each, have to spread over the banks.
  static constexpr int kSpread = kOperandRows >= 128 ? 3 : kOperandRows / 32 - 1;

  static __device__ __forceinline__ int unit(int part, int row_or_k, int chunk) {
    if constexpr (kByColumns) {
      return (part * G::kDepth + row_or_k) * kAcross + (chunk ^ ((row_or_k & kSpread) << 2));
    } else {
      return (part * kOperandRows + row_or_k) * G::kPitch + G::swizzled(row_or_k, chunk);
    }
  }

  // By columns a thread's chunks are of the same eight rows.
  static_assert(!kByColumns || G::kThreads % kAcross == 0, "whole k a chunk");
  static constexpr int kScales = !G::Format::kScaled ? 0 : kByColumns ? 8 : kPer;

  u4 value[kPer][sizeof(T) / 2];
  float scale[kScales ? kScales : 1];
  const Matrix& m;
  const T* base[kByColumns ? 1 : kPer];
  int64_t row0;

  // Chunk c of this thread: its row and chunk along k, or its k and chunk along the rows.
  static __device__ __forceinline__ int line(int c) {
    return (threadIdx.x + c * G::kThreads) / (kByColumns ? kAcross : G::kChunks);
  }
  static __device__ __forceinline__ int place(int c) {
    return (threadIdx.x + c * G::kThreads) % (kByColumns ? kAcross : G::kChunks);
  }

  __device__ __forceinline__ Stager(const Matrix& matrix, int64_t first_row) : m(matrix), row0(first_row) {
    if constexpr (!kByColumns) {
#pragma unroll
      for (int c = 0; c < kPer; ++c) {
        const int r = line(c);
        const void* matrix_base = m.first;
        int64_t row = row0 + r;
        if constexpr (kSource == kPairedRows) {
          row = row0 + paired_feature<G>(r);
          if (paired_second<G>(r)) matrix_base = m.second;
        }
        row = min(row, m.rows - 1);
        base[c] = static_cast<const T*>(matrix_base) + row * m.ld + place(c) * 8;
        if constexpr (G::Format::kScaled) {
          const bool second = kSource == kPairedRows && paired_second<G>(r);
          scale[c] = power_of_two(shift_of((second ? m.second_top : m.top)[row]));
        }
      }
    } else if constexpr (G::Format::kScaled) {
#pragma unroll
      for (int i = 0; i < 8; ++i) scale[i] = power_of_two(shift_of(m.top[min(row0 + place(0) * 8 + i, m.rows - 1)]));
    }
  }

  static __device__ __forceinline__ void load(u4 (&v)[sizeof(T) / 2], const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v[i] = load_loose<u4>(p + i * (16 / sizeof(T)));
  }
  // The first `count` of 8 values, zeros after them.
  static __device__ __forceinline__ void load_some(u4 (&v)[sizeof(T) / 2], const T* p, int64_t count) {
    T some[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) some[i] = i < count ? p[i] : static_cast<T>(0.0f);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      v[i] = *reinterpret_cast<const u4*>(some + i * (16 / sizeof(T)));
    }
  }

  __device__ __forceinline__ void fetch(int64_t k0) {
    if constexpr (!kByColumns) {
      if (k0 + G::kDepth <= m.depth) {
#pragma unroll
        for (int c = 0; c < kPer; ++c) load(value[c], base[c] + k0);
      } else {
#pragma unroll
        for (int c = 0; c < kPer; ++c) load_some(value[c], base[c] + k0, m.depth - k0 - place(c) * 8);
      }
    } else {
      const void* from = m.first;
      int64_t at = k0, end = m.depth;
      if constexpr (kSource == kPairedColumns) {  // a step lies in one half: half is a multiple of it
        if (k0 >= m.half) {
          from = m.second;
          at = k0 - m.half;
        }
        end = m.segment;
      }
      const T* const corner = static_cast<const T*>(from) + at * m.ld + row0;
      const unsigned ld = static_cast<unsigned>(m.ld);  // 32-bit offsets: kMostColumns
      if (at + G::kDepth <= end && row0 + kOperandRows <= m.rows) {
#pragma unroll
        for (int c = 0; c < kPer; ++c) load(value[c], corner + (line(c) * ld + place(c) * 8));
      } else {
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
          load_some(value[c], corner + (line(c) * ld + place(c) * 8),
                    at + line(c) < end ? m.rows - row0 - place(c) * 8 : 0);
        }
      }
    }
  }

  __device__ __forceinline__ void stage(u4* buffer) const {
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      if constexpr (G::kParts == 1) {
        buffer[unit(0, line(c), place(c))] = value[c][0];
      } else if constexpr (G::Format::kScaled) {
        u4 part[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned a = value[c][i / 2][i % 2 * 2], b = value[c][i / 2][i % 2 * 2 + 1];
          unsigned hi, lo;
          split_half_pair(__builtin_bit_cast(float, a) * scale[kByColumns ? 2 * i : c],
                          __builtin_bit_cast(float, b) * scale[kByColumns ? 2 * i + 1 : c], hi, lo);
          part[0][i] = hi;
          part[1][i] = lo;
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) buffer[unit(p, line(c), place(c))] = part[p];
      } else {
        u4 part[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned a = value[c][i / 2][i % 2 * 2], b = value[c][i / 2][i % 2 * 2 + 1];
          unsigned hi, mid, lo;
          split_pair(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b), hi, mid, lo);
          part[0][i] = hi;
          part[1][i] = mid;
          part[2][i] = lo;
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) buffer[unit(p, line(c), place(c))] = part[p];
      }
    }
  }

  // k 16 t + 8 (lane / 32) .. + 7 of row first + lane % 32 (first a multiple of 32).
  static __device__ __forceinline__ u4 operand(const u4* buffer, int part, int first, int t) {
    const int lane = threadIdx.x % kWave;
    if constexpr (!kByColumns) {
      return buffer[unit(part, first + lane % 32, 2 * t + lane / 32)];
    } else {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4 lds_s4;
      const int k = lane / 32 * 8 + lane % 16 / 4;
      const int chunk = first / 8 + lane % 32 / 16 * 2 + lane % 4 / 2;
      u2 half[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = 2 * unit(part, 16 * t + k + 4 * h, chunk) + lane % 2;  // in 8 bytes
        half[h] = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(
            reinterpret_cast<const u2*>(buffer) + at)));
      }
      return u4{half[0][0], half[0][1], half[1][0], half[1][1]};
    }
  }
};

template <typename Format>
__device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
  if constexpr (Format::kScaled) {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  }
}

// The products of 16 k of the scaled format: what has a lo apart, 2^11 too large.
template <typename G>
__device__ __forceinline__ void scaled_products(const u4 (&fa)[2][G::kBlocksM], const u4 (&fb)[2][G::kBlocksN],
                                                f16v (&acc)[G::kBlocksM][G::kBlocksN],
                                                f16v (&low)[G::kBlocksM][G::kBlocksN]) {
  typedef typename G::Format Format;
#pragma unroll
  for (int q = 0; q < Format::kProducts; ++q) {
#pragma unroll
    for (int i = 0; i < G::kBlocksM; ++i) {
#pragma unroll
      for (int j = 0; j < G::kBlocksN; ++j) {
        f16v& sum = q < 2 ? low[i][j] : acc[i][j];
        sum = mfma<Format>(fa[Format::part_a(q)][i], fb[Format::part_b(q)][j], sum);
      }
    }
  }
}
template <typename G>
__device__ __forceinline__ void add_low(f16v (&acc)[G::kBlocksM][G::kBlocksN],
                                        const f16v (&low)[G::kBlocksM][G::kBlocksN]) {
#pragma unroll
  for (int i = 0; i < G::kBlocksM; ++i) {
#pragma unroll
    for (int j = 0; j < G::kBlocksN; ++j) acc[i][j] += low[i][j] * 0x1p-11f;
  }
}

// Accumulates rows x columns of a tile over `steps` depth steps from k0. Two LDS buffers: while
// one is multiplied the next step's registers go into the other, and the step after that is
// fetched, so one barrier a step is enough.
template <typename G, typename A, typename B>
__device__ __forceinline__ void multiply(u4* lds, A& a, B& b, int64_t k0, int64_t steps,
                                         f16v (&acc)[G::kBlocksM][G::kBlocksN]) {
  constexpr int kBuffer = A::kUnits + B::kUnits;
  const int wave = threadIdx.x / kWave;
  const int row_a = wave / G::kWavesN * G::kWaveM, row_b = wave % G::kWavesN * G::kWaveN;
  typedef typename G::Format Format;
  f16v low[Format::kScaled ? G::kBlocksM : 1][Format::kScaled ? G::kBlocksN : 1] = {};
  a.fetch(k0);
  b.fetch(k0);
  a.stage(lds);
  b.stage(lds + A::kUnits);
  if (steps > 1) {
    a.fetch(k0 + G::kDepth);
    b.fetch(k0 + G::kDepth);
  }
  __syncthreads();
  for (int64_t s = 0; s < steps; ++s) {
    const u4* const now = lds + (s & 1) * kBuffer;
    if (s + 1 < steps) {
      u4* const next = lds + ((s + 1) & 1) * kBuffer;
      a.stage(next);
      b.stage(next + A::kUnits);
      if (s + 2 < steps) {
        a.fetch(k0 + (s + 2) * G::kDepth);
        b.fetch(k0 + (s + 2) * G::kDepth);
      }
    }
#pragma unroll
    for (int t = 0; t < G::kDepth / 16; ++t) {
      u4 fa[G::kParts][G::kBlocksM], fb[G::kParts][G::kBlocksN];
#pragma unroll
      for (int p = 0; p < G::kParts; ++p) {
#pragma unroll
        for (int i = 0; i < G::kBlocksM; ++i) fa[p][i] = A::operand(now, p, row_a + 32 * i, t);
#pragma unroll
        for (int j = 0; j < G::kBlocksN; ++j) fb[p][j] = B::operand(now + A::kUnits, p, row_b + 32 * j, t);
      }
      if constexpr (Format::kScaled) {
        scaled_products<G>(fa, fb, acc, low);
      } else if constexpr (G::kShortSums) {
#pragma unroll
        for (int i = 0; i < G::kBlocksM; ++i) {
#pragma unroll
          for (int j = 0; j < G::kBlocksN; ++j) {
            f16v sum = {};
#pragma unroll
            for (int q = 0; q < Format::kProducts; ++q) {
              sum = mfma<Format>(fa[Format::part_a(q)][i], fb[Format::part_b(q)][j], sum);
            }
            acc[i][j] += sum;
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < Format::kProducts; ++q) {
#pragma unroll
          for (int i = 0; i < G::kBlocksM; ++i) {
#pragma unroll
            for (int j = 0; j < G::kBlocksN; ++j) {
              acc[i][j] = mfma<Format>(fa[Format::part_a(q)][i], fb[Format::part_b(q)][j], acc[i][j]);
            }
          }
        }
      }
    }
    __syncthreads();
  }
  if constexpr (Format::kScaled) add_low<G>(acc, low);
}

// ---- direct staging -----------------------------------------------------------------------------
//
// bfloat16 operands whose rows are whole 16 bytes, and operands that were split before (kPlanes), go
// from memory to LDS without passing through registers (buffer loads with an LDS destination). The LDS
// layout is the Stager's: a wave's load fills 64 consecutive units, so the exclusive or goes into the
// lanes' source addresses. What lies outside a matrix is fetched from a place outside the buffer, which
// the hardware gives as zeros.
template <typename G, Source kSource, int kOperandRows>
struct Direct {
  typedef std::conditional_t<G::Format::kScaled, _Float16, __bf16> T;  // of a part
  typedef Stager<G, kSource, kOperandRows> Layout;
  static constexpr bool kByColumns = Layout::kByColumns;
  static constexpr int kPer = Layout::kPer, kUnits = Layout::kUnits, kPartUnits = kUnits / G::kParts;
  static constexpr int kLines = G::kThreads / (kByColumns ? Layout::kAcross : G::kChunks);  // of one load
  static constexpr unsigned kNowhere = 0x80000000u;
  static_assert(G::kParts < 3 && kPer * G::kThreads == kPartUnits, "every unit is loaded once");
  static_assert(kByColumns || (G::kSwizzled && kLines % 16 == 0), "a thread's chunk is the same in every load");
  static_assert(kSource != kPairedRows || G::kWaveN / 2 % (kWave / G::kChunks) == 0, "a wave's rows are of one matrix");

  const Matrix& m;
  int64_t row0;
  unsigned offset[kPer];  // bytes from the tile's corner
  int chunk, wave;

  __device__ __forceinline__ Direct(const Matrix& matrix, int64_t first_row) : m(matrix), row0(first_row) {
    const unsigned ld = static_cast<unsigned>(m.ld);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    chunk = G::swizzled(Layout::line(0), Layout::place(0));
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const int line = Layout::line(c);
      if constexpr (kByColumns) {
        const int column = (Layout::place(c) ^ ((line & Layout::kSpread) << 2)) * 8;
        offset[c] = row0 + column < m.rows ? (line * ld + column) * sizeof(T) : kNowhere;
      } else {
        const int r = kSource == kPairedRows ? paired_feature<G>(line) : line;
        offset[c] = row0 + r < m.rows ? (r * ld + chunk * 8) * sizeof(T) : kNowhere;
      }
    }
  }

  // The depth step at k0 into `buffer`; zeros from k_end on.
  __device__ __forceinline__ void fetch(u4* buffer, int64_t k0, int64_t k_end) const {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) void lds_void;
    constexpr int64_t kMost = 0x7fffffff;  // offsets are below it, kNowhere above
    const auto buffer_at = [](const T* p, int64_t bytes) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, static_cast<int>(min(bytes, kMost)), 0x00027000);
    };
    if constexpr (kByColumns) {
      const void* from = m.first;
      int64_t at = k0, end = m.depth;
      if constexpr (kSource == kPairedColumns) {
        if (k0 >= m.half) {
          from = m.second;
          at = k0 - m.half;
        }
        end = m.segment;
      }
      const int64_t bytes = k0 < k_end && at < end ? ((end - at) * m.ld - row0) * static_cast<int64_t>(sizeof(T)) : 0;
#pragma unroll
      for (int p = 0; p < G::kParts; ++p) {
        const auto source = buffer_at(static_cast<const T*>(from) + p * m.part + at * m.ld + row0, bytes);
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              source, (lds_void*)(buffer + p * kPartUnits + c * G::kThreads + wave * kWave), 16, offset[c], 0, 0, 0);
        }
      }
    } else {
      const int64_t corner = row0 * m.ld + k0;
      const unsigned beyond = k0 + chunk * 8 < min(m.depth, k_end) ? 0 : kNowhere;
#pragma unroll
      for (int p = 0; p < G::kParts; ++p) {
        const auto first = buffer_at(static_cast<const T*>(m.first) + p * m.part + corner, kMost);
        const auto second = kSource == kPairedRows
                                ? buffer_at(static_cast<const T*>(m.second) + p * m.part + corner, kMost) : first;
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
          const int line = c * kLines + (G::kWaveN / 2 % kLines == 0 ? 0 : wave * (kWave / G::kChunks));
          const bool up = kSource == kPairedRows && paired_second<G>(line);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              up ? second : first, (lds_void*)(buffer + p * kPartUnits + c * G::kThreads + wave * kWave), 16,
              offset[c] | beyond, 0, 0, 0);
        }
      }
    }
#endif
  }

  static __device__ __forceinline__ u4 operand(const u4* buffer, int part, int first, int t) {
    return Layout::operand(buffer, part, first, t);
  }
};

// multiply() for direct staging. A step's operands of 16 k are read while the 16 k before are
// multiplied; the barrier comes before a step's last products, whose operands are in registers, so
// the buffer can be filled again (for the step after the next) while they run.
template <typename G, typename A, typename B>
struct DirectProduct {
  static constexpr int kParts16 = G::kDepth / 16;
  static constexpr int kProducts = G::kBlocksM * G::kBlocksN;
  static constexpr int kReads = G::kBlocksM * (A::kByColumns ? 2 : 1) + G::kBlocksN * (B::kByColumns ? 2 : 1);
  static_assert(kParts16 % 2 == 0, "operand registers take turns");
  const A& a;
  const B& b;
  int row_a, row_b;
  int64_t k_end;
  u4 fa[2][G::kBlocksM], fb[2][G::kBlocksN];
  f16v (&acc)[G::kBlocksM][G::kBlocksN];

  __device__ __forceinline__ void read(const u4* from_a, const u4* from_b, int t) {
#pragma unroll
    for (int i = 0; i < G::kBlocksM; ++i) fa[t % 2][i] = A::operand(from_a, 0, row_a + 32 * i, t);
#pragma unroll
    for (int j = 0; j < G::kBlocksN; ++j) fb[t % 2][j] = B::operand(from_b, 0, row_b + 32 * j, t);
  }
  __device__ __forceinline__ void products(int t) {
#pragma unroll
    for (int i = 0; i < G::kBlocksM; ++i) {
#pragma unroll
      for (int j = 0; j < G::kBlocksN; ++j) acc[i][j] = mfma<Bf16>(fa[t % 2][i], fb[t % 2][j], acc[i][j]);
    }
  }
  // Instruction order: two LDS reads after each of the first products, loads spread over all.
  template <int kLoads>
  static __device__ __forceinline__ void order() {
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (2 * i < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      if ((i + 1) * kLoads / kProducts > i * kLoads / kProducts) {
        __builtin_amdgcn_sched_group_barrier(0x020, (kLoads + kProducts - 1) / kProducts, 0);
      }
    }
  }
  // One depth step: `now` is multiplied and then takes the step at k2; `next`'s first operands are
  // read.
  __device__ __forceinline__ void step(u4* now_a, u4* now_b, const u4* next_a, const u4* next_b, int64_t k2) {
#pragma unroll
    for (int t = 0; t + 1 < kParts16; ++t) {
      read(now_a, now_b, t + 1);
      products(t);
      order<0>();
    }
    __syncthreads();
    a.fetch(now_a, k2, k_end);
    b.fetch(now_b, k2, k_end);
    read(next_a, next_b, 0);
    products(kParts16 - 1);
    order<A::kPer + B::kPer>();
  }
};

// The buffers are arrays of their own, so that the compiler can tell a load into one from the reads
// of the other and waits only at the barriers. Steps come in pairs: one past the end is zeros.
template <typename G, typename A, typename B>
__device__ __forceinline__ void multiply(u4* a0, u4* b0, u4* a1, u4* b1, const A& a, const B& b, int64_t k0,
                                         int64_t steps, f16v (&acc)[G::kBlocksM][G::kBlocksN]) {
  const int wave = threadIdx.x / kWave;
  const int64_t k_end = k0 + steps * G::kDepth;
  DirectProduct<G, A, B> p{a, b, wave / G::kWavesN * G::kWaveM, wave % G::kWavesN * G::kWaveN, k_end, {}, {}, acc};
  a.fetch(a0, k0, k_end);
  b.fetch(b0, k0, k_end);
  __syncthreads();
  a.fetch(a1, k0 + G::kDepth, k_end);
  b.fetch(b1, k0 + G::kDepth, k_end);
  p.read(a0, b0, 0);
  for (int64_t s = 0; s < steps; s += 2) {
    p.step(a0, b0, a1, b1, k0 + (s + 2) * G::kDepth);
    p.step(a1, b1, a0, b0, k0 + (s + 3) * G::kDepth);
  }
  __syncthreads();  // no load may arrive in LDS after the workgroup has ended
}

// Waits until all but this wave's last kLeft memory operations and all its LDS operations are done, then
// for the workgroup's other waves. (Operations end in their order; __syncthreads waits for all.)
template <int kLeft>
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
}

// multiply() for a second operand that was split before: its parts come into LDS directly, two steps
// ahead, into the third of three buffers; the first operand's next step, fetched a step before, is split
// into its buffer while a step is multiplied. A step issues kLoads of these direct loads whatever its
// place, so when it waits for all but its last kLoads operations the step before's have arrived.
// Two buffers with the loads one step ahead left part of their latency uncovered (dx of 65,536 x 1,024 x
// 2,731 350 TFLOP/s, now 376; weight gradients 317, now 338); the first operand a step further ahead
// gained nothing.
template <typename G, typename A, typename B>
struct PlanesProduct {
  static constexpr int kLoads = G::kParts * B::kPer;
  A& a;
  const B& b;
  int row_a, row_b;
  int64_t k_end;
  f16v (&acc)[G::kBlocksM][G::kBlocksN];
  f16v (&low)[G::kBlocksM][G::kBlocksN];

  __device__ __forceinline__ void step(const u4* now_a, const u4* now_b, u4* next_a, u4* after_b, int64_t k2) {
    a.stage(next_a);
    a.fetch(k2);
    b.fetch(after_b, k2, k_end);
#pragma unroll
    for (int t = 0; t < G::kDepth / 16; ++t) {
      u4 fa[2][G::kBlocksM], fb[2][G::kBlocksN];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < G::kBlocksM; ++i) fa[p][i] = A::operand(now_a, p, row_a + 32 * i, t);
#pragma unroll
        for (int j = 0; j < G::kBlocksN; ++j) fb[p][j] = B::operand(now_b, p, row_b + 32 * j, t);
      }
      scaled_products<G>(fa, fb, acc, low);
    }
    meet<kLoads>();
  }
};

// The buffers are arrays of their own, so that the compiler sees that a load into one is not what another's
// reads wait for.
template <typename G, typename A, typename B>
__device__ __forceinline__ void multiply_planes(u4* a0, u4* b0, u4* a1, u4* b1, u4* a2, u4* b2, A& a, const B& b,
                                                int64_t k0, int64_t steps, f16v (&acc)[G::kBlocksM][G::kBlocksN]) {
  constexpr int64_t kDepth = G::kDepth;
  const int wave = threadIdx.x / kWave;
  f16v low[G::kBlocksM][G::kBlocksN] = {};
  PlanesProduct<G, A, B> p{a, b, wave / G::kWavesN * G::kWaveM, wave % G::kWavesN * G::kWaveN, k0 + steps * kDepth, acc, low};
  b.fetch(b0, k0, p.k_end);
  b.fetch(b1, k0 + kDepth, p.k_end);
  a.fetch(k0);
  a.stage(a0);
  a.fetch(k0 + kDepth);
  meet<0>();
  for (int64_t s = 0; s < steps; s += 3) {
    p.step(a0, b0, a1, b2, k0 + (s + 2) * kDepth);
    if (s + 1 >= steps) break;
    p.step(a1, b1, a2, b0, k0 + (s + 3) * kDepth);
    if (s + 2 >= steps) break;
    p.step(a2, b2, a0, b1, k0 + (s + 4) * kDepth);
  }
  meet<0>();  // no load may arrive in LDS after the workgroup has ended
  add_low<G>(acc, low);
}

// How a tile's operands come into LDS: both through registers (split there), both directly, or the
// second, split before, directly.
enum Staging { kRegisters, kDirect, kPlanes };

// A tile's accumulators.
template <typename G, Staging kStaging, Source kSourceA, Source kSourceB>
__device__ __forceinline__ void accumulate(const Matrix& a, const Matrix& b, int64_t row0, int64_t column0,
                                           int64_t k0, int64_t steps, f16v (&acc)[G::kBlocksM][G::kBlocksN]) {
  if constexpr (kStaging == kDirect) {
    typedef Direct<G, kSourceA, G::kM> A;
    typedef Direct<G, kSourceB, G::kN> B;
    __shared__ u4 a0[A::kUnits], b0[B::kUnits], a1[A::kUnits], b1[B::kUnits];
    multiply<G>(a0, b0, a1, b1, A(a, row0), B(b, column0), k0, steps, acc);
  } else if constexpr (kStaging == kPlanes) {
    typedef Stager<G, kSourceA, G::kM> A;
    typedef Direct<G, kSourceB, G::kN> B;
    __shared__ u4 a0[A::kUnits], b0[B::kUnits], a1[A::kUnits], b1[B::kUnits], a2[A::kUnits], b2[B::kUnits];
    A stage_a(a, row0);
    multiply_planes<G>(a0, b0, a1, b1, a2, b2, stage_a, B(b, column0), k0, steps, acc);
  } else {
    typedef Stager<G, kSourceA, G::kM> A;
    typedef Stager<G, kSourceB, G::kN> B;
    __shared__ u4 lds[2 * (A::kUnits + B::kUnits)];
    A stage_a(a, row0);
    B stage_b(b, column0);
    multiply<G>(lds, stage_a, stage_b, k0, steps, acc);
  }
}

// HalfParts: what the results of a tile's rows and columns are scaled back by.
template <typename G>
struct Shifts {
  int row[G::Format::kScaled ? G::kM : 1];

  __device__ __forceinline__ void load(const Matrix& a, int64_t row0) {
    if constexpr (G::Format::kScaled) {
      for (int r = threadIdx.x; r < G::kM; r += G::kThreads) row[r] = -shift_of(a.top[min(row0 + r, a.rows - 1)]);
    }
  }
  static __device__ __forceinline__ int column(const unsigned* top, int64_t column) {
    if constexpr (G::Format::kScaled) return -shift_of(top[column]);
    return 0;
  }
  __device__ __forceinline__ float back(float v, int r, int column_shift) const {
    if constexpr (G::Format::kScaled) return __builtin_amdgcn_ldexpf(v, row[r] + column_shift);
    return v;
  }
};

// Workgroup -> tile. Consecutive workgroups go to the 8 XCDs in turn, each with its own L2: an
// XCD takes a run of consecutive tiles, in bands of 8 tile rows walked column by column, so that
// what runs on it at one time shares operand rows and columns.
struct TileAt {
  int64_t m, n;
};
__device__ __forceinline__ TileAt tile_at(int64_t tiles_m, int64_t tiles_n) {
  const unsigned total = static_cast<unsigned>(tiles_m * tiles_n), id = blockIdx.x;
  const unsigned xcd = id % 8, share = total / 8, rest = total % 8;
  const unsigned at = xcd * share + min(xcd, rest) + id / 8;
  const unsigned band_tiles = 8 * static_cast<unsigned>(tiles_n);
  const unsigned band = at / band_tiles, in_band = at % band_tiles;
  const unsigned height = min(static_cast<unsigned>(tiles_m) - band * 8, 8u);
  // The same for every lane, which the compiler does not see through the divisions.
  return {__builtin_amdgcn_readfirstlane(band * 8 + in_band % height),
          __builtin_amdgcn_readfirstlane(in_band / height)};
}

struct ForwardArgs {
  Matrix x, weights;
  const void *gate_bias, *up_bias;
  void* h;
  float* pre;
  int64_t rows, hidden, pre_pitch, tiles_m, tiles_n;
  int activation;
};

template <typename G, Staging kStaging>
__global__ __launch_bounds__(G::kThreads) void gated_forward_kernel(ForwardArgs args) {
  typedef typename G::T T;
  const TileAt tile = tile_at(args.tiles_m, args.tiles_n);
  const int64_t row0 = tile.m * G::kM, feature0 = tile.n * (G::kN / 2);
  __shared__ Shifts<G> shifts;
  shifts.load(args.x, row0);  // read after the product's barriers
  f16v acc[G::kBlocksM][G::kBlocksN] = {};
  accumulate<G, kStaging, kRows, kPairedRows>(args.x, args.weights, row0, feature0, 0,
                                             ceil_div(args.x.depth, G::kDepth), acc);

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  constexpr int kHalf = G::kBlocksN / 2;
  const int rows = static_cast<int>(min(args.rows - row0, static_cast<int64_t>(G::kM)));
  const int features = static_cast<int>(min(args.hidden - feature0, static_cast<int64_t>(G::kN / 2)));
  T* const h = static_cast<T*>(args.h) + row0 * args.hidden + feature0;
  float* const pre_g = args.pre + row0 * args.pre_pitch + feature0;
  float* const pre_u = pre_g + args.rows * args.pre_pitch;
  const unsigned hidden = static_cast<unsigned>(args.hidden), pitch = static_cast<unsigned>(args.pre_pitch);
#pragma unroll
  for (int j = 0; j < kHalf; ++j) {
    const int feature = wave % G::kWavesN * (G::kWaveN / 2) + 32 * j + lane % 32;
    if (feature >= features) continue;
    const float gate_bias = args.gate_bias ? to_float(static_cast<const T*>(args.gate_bias)[feature0 + feature]) : 0.0f;
    const float up_bias = args.up_bias ? to_float(static_cast<const T*>(args.up_bias)[feature0 + feature]) : 0.0f;
    const int shift_g = Shifts<G>::column(args.weights.top, feature0 + feature);
    const int shift_u = Shifts<G>::column(args.weights.second_top, feature0 + feature);
#pragma unroll
    for (int i = 0; i < G::kBlocksM; ++i) {
      const int first = wave / G::kWavesN * G::kWaveM + 32 * i + lane / 32 * 4;
      const unsigned at_h = first * hidden + feature, at_pre = first * pitch + feature;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int down = r % 4 + 8 * (r / 4);
        if (first + down >= rows) continue;
        const float g = shifts.back(acc[i][j][r], first + down, shift_g) + gate_bias;
        const float u = shifts.back(acc[i][j + kHalf][r], first + down, shift_u) + up_bias;
        // Past the caches: every CU writes its tile at about the same time, and a burst of 84 MB
        // that waits in the L2s holds up the next tiles' loads (16,384 x 2,048 x 8,192 bfloat16:
        // 1,249 us with plain stores, 1,106 with these).
        __builtin_nontemporal_store(from_float<T>(activate(args.activation, g).value * u), &h[at_h + down * hidden]);
        if (args.pre) {
          __builtin_nontemporal_store(g, &pre_g[at_pre + down * pitch]);
          __builtin_nontemporal_store(u, &pre_u[at_pre + down * pitch]);
        }
      }
    }
  }
}

// ---- few rows -----------------------------------------------------------------------------------
//
// Up to 32 rows the weights' bytes bound the forward, and what counts is how many of them are on
// their way. A workgroup takes 16 or 32 features (their gate and up rows), its waves every fourth or
// eighth 128 bytes of the rows, straight from memory into matrix operands of 16 x 16 x 32 products;
// nothing passes through LDS but the waves' sums at the end. 16 rows, 4,096 x 10,240 bfloat16: 39.7
// us, 4.2 TB/s (32 features and 8 waves: 47.8); 4,096 x 5,120 float32, whose operands are split in
// registers: 46.2 with 32 features and 8 waves, which share the split rows of x (16 and 4: 50.8).
// Small layers want more waves: 1 row, 256 x 683 float32, 3.3 us with 8 waves, 4.0 with 4.
template <typename T>
struct Step {
  typedef std::conditional_t<std::is_same_v<T, float>, Bf16Parts, Bf16> Format;
  static constexpr int kDepth = 128 / static_cast<int>(sizeof(T));  // 64 bfloat16 or 32 float32
  static constexpr int kChunks = kDepth / 32;                      // of 8 values a lane
  u4 value[kChunks][sizeof(T) / 2];

  __device__ __forceinline__ void load(const T* row, int64_t k, int64_t width) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int64_t at = k + 32 * c;
      if (at + 8 <= width) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
          value[c][i] = load_loose<u4>(row + at + i * (16 / sizeof(T)));
        }
      } else {
        T some[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) some[i] = at + i < width ? row[at + i] : static_cast<T>(0.0f);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
          value[c][i] = *reinterpret_cast<const u4*>(some + i * (16 / sizeof(T)));
        }
      }
    }
  }

  // Chunk c's operand parts.
  __device__ __forceinline__ void parts(int c, u4 (&part)[Format::kParts]) const {
    if constexpr (Format::kParts == 1) {
      part[0] = value[c][0];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned a = value[c][i / 2][i % 2 * 2], b = value[c][i / 2][i % 2 * 2 + 1];
        unsigned hi, mid, lo;
        split_pair(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b), hi, mid, lo);
        part[0][i] = hi;
        part[1][i] = mid;
        part[2][i] = lo;
      }
    }
  }
};

constexpr int kFewRows = 32;  // 64 rows, 4,096 x 10,240 bfloat16: 71 us, and 57 with the smallest tiles

template <typename T, int kBlocks, int kPairs, int kWaves>  // kBlocks of 16 rows, kPairs of 16 features
__global__ __launch_bounds__(kWaves * kWave) void gated_few_rows_kernel(ForwardArgs args) {
  typedef typename Step<T>::Format Format;
  constexpr int kParts = Format::kParts, kThreads = kWaves * kWave, kTiles = 2 * kPairs;
  constexpr int kFewFeatures = 16 * kPairs;
  __shared__ f4 sums[kWaves][kBlocks][kTiles][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t feature0 = static_cast<int64_t>(blockIdx.x) * kFewFeatures, width = args.x.depth;
  const T *weight[kTiles], *row[kBlocks];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {  // the gate's, then up's
    weight[t] = static_cast<const T*>(t < kPairs ? args.weights.first : args.weights.second) +
                min(feature0 + t % kPairs * 16 + lane % 16, args.hidden - 1) * width;
  }
#pragma unroll
  for (int m = 0; m < kBlocks; ++m) {
    row[m] = static_cast<const T*>(args.x.first) + min(static_cast<int64_t>(16 * m + lane % 16), args.rows - 1) * width;
  }
  f4 acc[kBlocks][kTiles] = {};
  Step<T> b[kTiles], a[kBlocks];
  const int64_t steps = ceil_div(width, Step<T>::kDepth);
  const auto fetch = [&](int64_t s) {
    const int64_t k = s * Step<T>::kDepth + lane / 16 * 8;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) b[t].load(weight[t], k, width);
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) a[m].load(row[m], k, width);
  };
  if (wave < steps) fetch(wave);
  for (int64_t s = wave; s < steps; s += kWaves) {
#pragma unroll
    for (int c = 0; c < Step<T>::kChunks; ++c) {
      u4 pa[kBlocks][kParts];
#pragma unroll
      for (int m = 0; m < kBlocks; ++m) a[m].parts(c, pa[m]);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        u4 pb[kParts];
        b[t].parts(c, pb);
#pragma unroll
        for (int q = 0; q < Format::kProducts; ++q) {
#pragma unroll
          for (int m = 0; m < kBlocks; ++m) {
            acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf8, pa[m][Format::part_a(q)]),
                __builtin_bit_cast(bf8, pb[Format::part_b(q)]), acc[m][t], 0, 0, 0);
          }
        }
      }
    }
    if (s + kWaves < steps) fetch(s + kWaves);
  }
#pragma unroll
  for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t) sums[wave][m][t][lane] = acc[m][t];
  }
  __syncthreads();
  // Result (row 16 m + 4 (lane / 16) + r, feature lane % 16 of its block) lies in element r of lane.
  for (int e = threadIdx.x; e < 16 * kBlocks * kFewFeatures; e += kThreads) {
    const int f = e % kFewFeatures, r = e / kFewFeatures;
    const int64_t feature = feature0 + f;
    if (r >= args.rows || feature >= args.hidden) continue;
    const int from = r % 16 / 4 * 16 + f % 16;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      g += sums[w][r / 16][f / 16][from][r % 4];
      u += sums[w][r / 16][kPairs + f / 16][from][r % 4];
    }
    if (args.gate_bias) g += to_float(static_cast<const T*>(args.gate_bias)[feature]);
    if (args.up_bias) u += to_float(static_cast<const T*>(args.up_bias)[feature]);
    static_cast<T*>(args.h)[r * args.hidden + feature] = from_float<T>(activate(args.activation, g).value * u);
    if (args.pre) {
      args.pre[r * args.pre_pitch + feature] = g;
      args.pre[(args.rows + r) * args.pre_pitch + feature] = u;
    }
  }
}

// ---- few tiles, float32 -------------------------------------------------------------------------
//
// A float32 layer with few tiles for the 256 CUs is bound by a workgroup's chain of steps: loads,
// split, LDS, barrier, products, some 1.1 us for each 16 of the depth whichever tile is taken. Here a
// workgroup takes 32 rows of 32 features, and its eight waves every eighth 16 of the depth, from
// memory straight into operands (each wave splits what it multiplies, so nothing is split once for
// several), so the chain is an eighth as long; their sums meet in LDS once at the end. Measured, this
// kernel, the 64 x 64 tiles of Bf16Parts, those of HalfParts without their scales' two launches, us:
// 64 x 256 x 683 (44 workgroups) 8.0, 17.8, 12.2; 100 x 1,024 x 1,024 (128) 20.0, 52.4, 31.7;
// 128 x 2,048 x 2,048 (256) 38.9, 99.7, 58.2; 256 x 512 x 1,365 (344) 22.5, 29.6, 18.9; 1,000 x 512 x
// 1,365 (1,376) 59.4, 41.2, 24.4. It is taken up to a workgroup a CU; the gain ends above that.
constexpr int kShortWaves = 8, kShortSide = 32;

__device__ __forceinline__ void load_eight(f4 (&v)[2], const float* row, int64_t k, int64_t width) {
  if (k + 8 <= width) {
    v[0] = load_loose<f4>(row + k);
    v[1] = load_loose<f4>(row + k + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = k + i < width ? row[k + i] : 0.0f;
  }
}

__device__ __forceinline__ void split_eight(const f4 (&v)[2], u4 (&part)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned hi, mid, lo;
    split_pair(v[i / 2][i % 2 * 2], v[i / 2][i % 2 * 2 + 1], hi, mid, lo);
    part[0][i] = hi;
    part[1][i] = mid;
    part[2][i] = lo;
  }
}

__global__ __launch_bounds__(kShortWaves * kWave, 4) void gated_short_kernel(ForwardArgs args) {
  typedef Bf16Parts Format;
  __shared__ f4 sums[kShortWaves][2][4][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kShortSide, feature0 = static_cast<int64_t>(blockIdx.x) * kShortSide;
  const int64_t width = args.x.depth, feature = min(feature0 + lane % 32, args.hidden - 1);
  const float* const from[3] = {
      static_cast<const float*>(args.x.first) + min(row0 + lane % 32, args.rows - 1) * width,
      static_cast<const float*>(args.weights.first) + feature * width,
      static_cast<const float*>(args.weights.second) + feature * width};
  f16v acc[2] = {};
  f4 value[2][3][2];
  const int64_t steps = ceil_div(width, 16);
  const auto fetch = [&](int64_t s, int set) {
#pragma unroll
    for (int m = 0; m < 3; ++m) load_eight(value[set][m], from[m], 16 * s + lane / 32 * 8, width);
  };
#pragma unroll
  for (int set = 0; set < 2; ++set) {
    if (wave + set * kShortWaves < steps) fetch(wave + set * kShortWaves, set);
  }
  for (int64_t s0 = wave; s0 < steps; s0 += 2 * kShortWaves) {
#pragma unroll
    for (int set = 0; set < 2; ++set) {
      const int64_t s = s0 + set * kShortWaves;
      if (s >= steps) break;
      u4 part[3][3];
#pragma unroll
      for (int m = 0; m < 3; ++m) split_eight(value[set][m], part[m]);
      if (s + 2 * kShortWaves < steps) fetch(s + 2 * kShortWaves, set);
#pragma unroll
      for (int q = 0; q < Format::kProducts; ++q) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[j] = mfma<Format>(part[0][Format::part_a(q)], part[1 + j][Format::part_b(q)], acc[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sums[wave][j][r][lane] = f4{acc[j][4 * r], acc[j][4 * r + 1], acc[j][4 * r + 2], acc[j][4 * r + 3]};
    }
  }
  __syncthreads();
  // Row r and feature f of the tile: element r % 4 of quad r / 8, lane f + 32 for every second four rows.
  for (int e = threadIdx.x; e < 32 * 32; e += kShortWaves * kWave) {
    const int f = e % 32, r = e / 32;
    const int64_t row = row0 + r, at = feature0 + f;
    if (row >= args.rows || at >= args.hidden) continue;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < kShortWaves; ++w) {
      g += sums[w][0][r / 8][f + r / 4 % 2 * 32][r % 4];
      u += sums[w][1][r / 8][f + r / 4 % 2 * 32][r % 4];
    }
    if (args.gate_bias) g += static_cast<const float*>(args.gate_bias)[at];
    if (args.up_bias) u += static_cast<const float*>(args.up_bias)[at];
    static_cast<float*>(args.h)[row * args.hidden + at] = activate(args.activation, g).value * u;
    if (args.pre) {
      args.pre[row * args.pre_pitch + at] = g;
      args.pre[(args.rows + row) * args.pre_pitch + at] = u;
    }
  }
}

// A product's results: rows x columns at out[row ld + column], or with `partials` the sum over
// one of gridDim.y runs of the depth, [run][rows][columns]. Rows from `half` on are those of a
// second matrix (the weight gradients); the `segment` first rows of each exist.
struct ProductArgs {
  Matrix a, b;
  void *first, *second;
  float* partials;
  int64_t rows, columns, half, segment, tiles_m, tiles_n, steps;
};

template <typename G, Staging kStaging, Source kSourceA, Source kSourceB>
__global__ __launch_bounds__(G::kThreads) void product_kernel(ProductArgs args) {
  typedef typename G::T T;
  const TileAt tile = tile_at(args.tiles_m, args.tiles_n);
  const int64_t row0 = tile.m * G::kM, column0 = tile.n * G::kN;
  const int64_t step0 = args.steps * blockIdx.y / gridDim.y, step1 = args.steps * (blockIdx.y + 1) / gridDim.y;
  __shared__ Shifts<G> shifts;
  shifts.load(args.a, row0);  // read after the product's barriers
  f16v acc[G::kBlocksM][G::kBlocksN] = {};
  accumulate<G, kStaging, kSourceA, kSourceB>(args.a, args.b, row0, column0, step0 * G::kDepth, step1 - step0, acc);

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int rows = static_cast<int>(min(args.rows - row0, static_cast<int64_t>(G::kM)));
  const int columns = static_cast<int>(min(args.columns - column0, static_cast<int64_t>(G::kN)));
  const unsigned ld = static_cast<unsigned>(args.columns);
#pragma unroll
  for (int i = 0; i < G::kBlocksM; ++i) {
    // A block's 32 rows are all in one half: halves are multiples of 64 rows.
    const int first = wave / G::kWavesN * G::kWaveM + 32 * i;
    const bool second = row0 + first >= args.half;
    const int64_t in_half = row0 + first - (second ? args.half : 0);
    const int there = static_cast<int>(min(args.segment - in_half, static_cast<int64_t>(32)));
    T* const out = static_cast<T*>(second ? args.second : args.first) + in_half * args.columns + column0;
    float* const partial = args.partials + (blockIdx.y * args.rows + row0 + first) * args.columns + column0;
#pragma unroll
    for (int j = 0; j < G::kBlocksN; ++j) {
      const int column = wave % G::kWavesN * G::kWaveN + 32 * j + lane % 32;
      if (column >= columns) continue;
      const unsigned at = lane / 32 * 4 * ld + column;
      const int shift = Shifts<G>::column(args.b.top, column0 + column);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int down = r % 4 + 8 * (r / 4);
        if (down + lane / 32 * 4 >= there || first + down + lane / 32 * 4 >= rows) continue;
        const float v = shifts.back(acc[i][j][r], first + down + lane / 32 * 4, shift);
        if (args.partials) partial[at + down * ld] = v;
        else out[at + down * ld] = from_float<T>(v);
      }
    }
  }
}

// Sum of the runs' partial results, in order, four columns a thread. Bound by their bytes
// (20,011 x 512, four runs: 27 us; one value a thread, with a division for each: 44).
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(ProductArgs args, int runs) {
  typedef T V __attribute__((ext_vector_type(4)));
  const int64_t quads = ceil_div(args.columns, 4), n = args.rows * args.columns, all = args.rows * quads;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < all; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = all >> 32 ? e / quads : static_cast<unsigned>(e) / static_cast<unsigned>(quads);
    const bool second = row >= args.half;
    const int64_t in_half = second ? row - args.half : row, column = 4 * (e - row * quads);
    if (in_half >= args.segment) continue;
    const float* const p = args.partials + row * args.columns + column;
    T* const out = static_cast<T*>(second ? args.second : args.first) + in_half * args.columns + column;
    if (column + 4 <= args.columns) {
      f4 sum = {};
#pragma unroll 4
      for (int run = 0; run < runs; ++run) sum += load_loose<f4>(p + run * n);
      V v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = from_float<T>(sum[i]);
      reinterpret_cast<Loose<V, T>*>(out)->v = v;
    } else {
      for (int i = 0; i < args.columns - column; ++i) {
        float sum = 0.0f;
        for (int run = 0; run < runs; ++run) sum += p[run * n + i];
        out[i] = from_float<T>(sum);
      }
    }
  }
}

// dg and du from dh, g and u, [rows][2 pitch] (zero between hidden and pitch), and their column
// sums over each workgroup's rows. A wave takes 256 features, four a lane, and every fourth row (kTops:
// every sixteenth, so that fewer workgroups end with an atomic for each column).
// kTops: also the largest magnitudes of the result's rows and columns, for HalfParts (maxima of bits:
// the order of the atomics does not matter). Bound by memory: 20 bytes a feature and row in float32
// (65,536 x 2,731: 770 us, 4.7 TB/s), 14 in bfloat16 (16,384 x 8,192: 380 us, 4.9 TB/s).
struct GateArgs {
  const void* grad_h;
  const float* pre;
  void* out;
  float* partials;  // [gridDim.y][2][pitch], or NULL
  unsigned *row_top, *column_top;  // kTops: [rows] and [2 pitch], zero before
  int64_t rows, hidden, pitch, rows_each;
  int activation;
};

__device__ __forceinline__ unsigned magnitude_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

template <bool kTops>
constexpr int kGateWaves = kTops ? 16 : 4;
template <typename T, bool kTops>
__global__ __launch_bounds__(kGateWaves<kTops> * kWave) void gate_backward_kernel(GateArgs args) {
  constexpr int kWaves = kGateWaves<kTops>;
  __shared__ f4 s_sum[2][kWaves][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t feature = static_cast<int64_t>(blockIdx.x) * 256 + 4 * lane;
  const int64_t end = min(args.rows, (blockIdx.y + 1) * args.rows_each);
  f4 gate_sum = {}, up_sum = {};
  u4 gate_top = {}, up_top = {};
  for (int64_t row = blockIdx.y * args.rows_each + wave; row < end; row += kWaves) {
    unsigned top = 0;
    if (feature < args.pitch) {
      const f4 g = *reinterpret_cast<const f4*>(args.pre + row * args.pitch + feature);
      const f4 u = *reinterpret_cast<const f4*>(args.pre + (args.rows + row) * args.pitch + feature);
      const T* const up = static_cast<const T*>(args.grad_h) + row * args.hidden + feature;
      typedef T V __attribute__((ext_vector_type(4)));
      f4 dh = {};
      if (feature + 4 <= args.hidden) {
        const V v = load_loose<V>(up);
#pragma unroll
        for (int i = 0; i < 4; ++i) dh[i] = to_float(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (feature + i < args.hidden) dh[i] = to_float(up[i]);
        }
      }
      f4 dg, du;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Activated a = activate(args.activation, g[i]);
        const bool inside = feature + i < args.hidden;
        const float to_gate = inside ? dh[i] * u[i] * a.slope : 0.0f, to_up = inside ? dh[i] * a.value : 0.0f;
        dg[i] = to_gate;
        du[i] = to_up;
        if constexpr (kTops) {
          gate_top[i] = max(static_cast<unsigned>(gate_top[i]), magnitude_bits(to_gate));
          up_top[i] = max(static_cast<unsigned>(up_top[i]), magnitude_bits(to_up));
          top = max(top, max(magnitude_bits(to_gate), magnitude_bits(to_up)));
        }
      }
      gate_sum += dg;
      up_sum += du;
      T* const out = static_cast<T*>(args.out) + row * 2 * args.pitch + feature;
      V vg, vu;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vg[i] = from_float<T>(dg[i]);
        vu[i] = from_float<T>(du[i]);
      }
      *reinterpret_cast<V*>(out) = vg;
      *reinterpret_cast<V*>(out + args.pitch) = vu;
    }
    if constexpr (kTops) {
      top = wave_max(top);
      if (lane == 0) atomicMax(args.row_top + row, top);
    }
  }
  if constexpr (kTops) {  // the waves' first: a sixteenth of the atomics
    s_sum[0][wave][lane] = __builtin_bit_cast(f4, gate_top);
    s_sum[1][wave][lane] = __builtin_bit_cast(f4, up_top);
    __syncthreads();
    if (wave < 2 && feature < args.pitch) {
      u4 top = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const u4 one = __builtin_bit_cast(u4, s_sum[wave][w][lane]);
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = max(static_cast<unsigned>(top[i]), static_cast<unsigned>(one[i]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) atomicMax(args.column_top + wave * args.pitch + feature + i, static_cast<unsigned>(top[i]));
    }
    __syncthreads();
  }
  if (!args.partials) return;
  s_sum[0][wave][lane] = gate_sum;
  s_sum[1][wave][lane] = up_sum;
  __syncthreads();
  if (wave < 2 && feature < args.pitch) {
    f4 total = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += s_sum[wave][w][lane];
    *reinterpret_cast<f4*>(args.partials + (2 * blockIdx.y + wave) * args.pitch + feature) = total;
  }
}

// Largest magnitudes (bits) of the rows or columns of up to three float32 matrices, into zeroed
// arrays. A workgroup takes 256 rows of 256 columns, a wave every sixteenth row, a lane four adjacent
// columns; the waves' column maxima meet in LDS first, for the fewest atomics (20,011 x 512 and two of
// 1,365 x 512: 17 us, with four waves to 64 rows 42; 65,536 x 1,024: 61 us, 4.4 TB/s).
struct TopJob {
  const float* matrix;
  int64_t rows, columns;
  unsigned *row_top, *column_top;  // either may be NULL
};
struct TopArgs {
  TopJob job[3];
  unsigned first[4];  // workgroups of the jobs before
  int count;
};
constexpr int kTopRows = 256, kTopColumns = 256, kTopWaves = 16;

__global__ __launch_bounds__(kTopWaves * kWave) void top_kernel(TopArgs args) {
  __shared__ u4 s_top[kTopWaves][kWave];
  int k = 0;
  while (k + 1 < args.count && blockIdx.x >= args.first[k + 1]) ++k;
  const TopJob& job = args.job[k];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const unsigned across = static_cast<unsigned>(ceil_div(job.columns, kTopColumns)), at = blockIdx.x - args.first[k];
  const int64_t row0 = static_cast<int64_t>(at / across) * kTopRows;
  const int64_t column = static_cast<int64_t>(at % across) * kTopColumns + 4 * lane;
  const int64_t end = min(row0 + kTopRows, job.rows);
  u4 tops = {};
#pragma unroll 8
  for (int64_t row = row0 + wave; row < end; row += kTopWaves) {
    const float* p = job.matrix + row * job.columns + column;
    float v[4] = {};
    if (column + 4 <= job.columns) {
      const f4 four = load_loose<f4>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = four[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (column + i < job.columns) v[i] = p[i];
      }
    }
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      tops[i] = max(static_cast<unsigned>(tops[i]), magnitude_bits(v[i]));
      top = max(top, magnitude_bits(v[i]));
    }
    if (job.row_top) {
      top = wave_max(top);
      if (lane == 0) atomicMax(job.row_top + row, top);
    }
  }
  if (!job.column_top) return;
  s_top[wave][lane] = tops;
  __syncthreads();
  if (wave >= 4) return;
  // Wave w takes value w of the lanes' four.
  unsigned top = 0;
#pragma unroll
  for (int w = 0; w < kTopWaves; ++w) top = max(top, static_cast<unsigned>(s_top[w][lane][wave]));
  if (column + wave < job.columns) atomicMax(job.column_top + column + wave, top);
}

template <typename T>
__global__ void zero_kernel(T* out, int64_t n) {
  for (int64_t k = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; k < n;
       k += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    out[k] = static_cast<T>(0.0f);
  }
}

// The two float16 parts of up to two float32 matrices, rows or columns scaled by their largest
// magnitude: [2][rows][ld], ld a multiple of 8 with zeros past the columns. A workgroup takes 32 rows
// of 512 columns, a wave every fourth row, a lane eight adjacent columns.
struct SplitJob {
  const float* matrix;
  int64_t rows, columns, ld;
  const unsigned *row_top, *column_top;  // one of them
  _Float16* out;
};
struct SplitArgs {
  SplitJob job[2];
  unsigned first[3];  // workgroups of the jobs before
};
constexpr int kSplitRows = 32, kSplitColumns = 512;

__global__ __launch_bounds__(256) void split_kernel(SplitArgs args) {
  const int k = blockIdx.x >= args.first[1];
  const SplitJob& job = args.job[k];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const unsigned across = static_cast<unsigned>(ceil_div(job.ld, kSplitColumns)), at = blockIdx.x - args.first[k];
  const int64_t row0 = static_cast<int64_t>(at / across) * kSplitRows;
  const int64_t column = static_cast<int64_t>(at % across) * kSplitColumns + 8 * lane;
  const int64_t end = min(row0 + kSplitRows, job.rows);
  if (column >= job.ld) return;
  float scale[8];
  if (job.column_top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) scale[i] = power_of_two(shift_of(job.column_top[min(column + i, job.columns - 1)]));
  }
#pragma unroll 4
  for (int64_t row = row0 + wave; row < end; row += 4) {
    f4 v[2];
    load_eight(v, job.matrix + row * job.columns, column, job.columns);
    if (job.row_top) {
      const float all = power_of_two(shift_of(job.row_top[row]));
#pragma unroll
      for (int i = 0; i < 8; ++i) scale[i] = all;
    }
    u4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned h, l;
      split_half_pair(v[i / 2][i % 2 * 2] * scale[2 * i], v[i / 2][i % 2 * 2 + 1] * scale[2 * i + 1], h, l);
      hi[i] = h;
      lo[i] = l;
    }
    *reinterpret_cast<u4*>(job.out + row * job.ld + column) = hi;
    *reinterpret_cast<u4*>(job.out + (job.rows + row) * job.ld + column) = lo;
  }
}

int launch_split(const SplitJob* jobs, int count, hipStream_t stream) {
  SplitArgs args{};
  int64_t groups = 0;
  for (int k = 0; k < 2; ++k) {
    args.first[k] = static_cast<unsigned>(groups);
    if (k >= count) continue;
    args.job[k] = jobs[k];
    groups += ceil_div(jobs[k].rows, kSplitRows) * ceil_div(jobs[k].ld, kSplitColumns);
  }
  args.first[2] = static_cast<unsigned>(groups);
  if (count == 1) args.first[1] = args.first[2];
  split_kernel<<<static_cast<unsigned>(groups), 256, 0, stream>>>(args);
  return check_launch("operand parts");
}

// Zeroes `zeros` floats at `all` (the jobs' arrays and others) and runs the jobs.
int launch_tops(unsigned* all, int64_t zeros, const TopJob* jobs, int count, hipStream_t stream) {
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(zeros, 256), 1024));
  zero_kernel<<<grid, 256, 0, stream>>>(reinterpret_cast<float*>(all), zeros);
  if (int status = check_launch("zero")) return status;
  TopArgs args{};
  args.count = count;
  int64_t groups = 0;
  for (int k = 0; k < count; ++k) {
    args.job[k] = jobs[k];
    args.first[k] = static_cast<unsigned>(groups);
    groups += ceil_div(jobs[k].rows, kTopRows) * ceil_div(jobs[k].columns, kTopColumns);
  }
  args.first[count] = static_cast<unsigned>(groups);
  top_kernel<<<static_cast<unsigned>(groups), kTopWaves * kWave, 0, stream>>>(args);
  return check_launch("largest magnitudes");
}

int zero(void* out, int64_t n, int dtype, hipStream_t stream) {
  if (!out || n == 0) return FHOAD_SUCCESS;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(n, 256), 4096));
  if (dtype == FHOAD_FLOAT32) zero_kernel<<<grid, 256, 0, stream>>>(static_cast<float*>(out), n);
  else zero_kernel<<<grid, 256, 0, stream>>>(static_cast<__bf16*>(out), n);
  return check_launch("zero");
}

// ---- host -------------------------------------------------------------------------------------

constexpr int kCus = 256;  // MI355X; on a device of fewer a plan is right as well, and less near the fastest
constexpr int64_t kPad = 64;  // features to a multiple of every tile's depth
int64_t padded(int64_t hidden) { return ceil_div(hidden, kPad) * kPad; }

// The tiles by type and size: 256 x 256 on eight waves where that gives every CU a workgroup,
// 128 x 128 on four, 64 x 64 on two for the smallest products. Eight waves of 64 x 128 results
// were the fastest shape (bfloat16 direct, input gradient at 16,384 x 2,048 x 8,192: 1,249 TFLOP/s;
// of 128 x 64: 1,104; four waves of 128 x 128: 1,138; 128 x 128 tiles, two workgroups a CU: 1,014).
template <typename Format> struct Tiles;
template <> struct Tiles<Bf16> {
  typedef Tile<Bf16, 256, 256, 4, 2, 64> Large;
  typedef Tile<Bf16, 128, 128, 2, 2, 64> Middle;
  typedef Tile<Bf16, 64, 64, 2, 1, 64> Small;
};
template <> struct Tiles<Bf16Parts> {
  typedef Tile<Bf16Parts, 256, 256, 2, 4, 16> Large;
  typedef Tile<Bf16Parts, 128, 128, 2, 2, 16> Middle;
  typedef Tile<Bf16Parts, 64, 64, 2, 1, 16, true> Small;
};
template <> struct Tiles<HalfParts> {
  typedef Tile<HalfParts, 128, 256, 2, 4, 32> Large;
  typedef Tile<HalfParts, 128, 128, 2, 2, 32> Middle;
  typedef Tile<HalfParts, 64, 64, 2, 1, 32> Small;
};

enum TileSize { kLarge, kMiddle, kSmall };

size_t align256(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Calls go(tile, staging) for the format, size and way of staging.
template <typename Format, typename TileType, typename Go>
void with_staging(Staging staging, Go go) {
  constexpr bool kWhole = std::is_same_v<Format, Bf16>, kSplit = std::is_same_v<TileType, Tiles<HalfParts>::Large>;
  if constexpr (kWhole || kSplit) {
    constexpr Staging kOther = kWhole ? kDirect : kPlanes;
    if (staging == kOther) {
      go(TileType{}, std::integral_constant<Staging, kOther>());
      return;
    }
  }
  go(TileType{}, std::integral_constant<Staging, kRegisters>());
}

// Whether a product of that many rows in HalfParts has its second operand split before: the large
// tiles, with rows enough to use each part often. Split by every workgroup on its way to LDS, 256 of
// the tile's 384 rows cost two thirds of the vector instructions beside the products. Inference in
// TFLOP/s, with and without: 65,536 x 1,024 x 2,731 330 and 286 (the kernel alone), 4,096 x 1,024 x 4,096
// 263 and 243, 2,000 x 1,024 x 2,731 175 and 170, 512 x 2,048 x 8,192 174 and 220.
bool split_before(TileSize size, int64_t rows) { return size == kLarge && rows >= 2048; }

// Values of a row of a split operand, and its two parts' bytes.
int64_t split_ld(int64_t columns) { return ceil_div(columns, 8) * 8; }
size_t split_bytes(int64_t rows, int64_t columns) { return align256(static_cast<size_t>(2 * rows * split_ld(columns)) * 2); }

// Splits the weights to `parts`, rows or columns scaled, and makes them the operand's matrices.
int split_weights(Matrix& operand, int64_t hidden, int64_t width, const unsigned* row_top, const unsigned* second_row_top,
                  const unsigned* column_top, char* parts, hipStream_t stream) {
  const int64_t ld = split_ld(width);
  _Float16 *const gate = reinterpret_cast<_Float16*>(parts), *const up = gate + 2 * hidden * ld;
  const SplitJob jobs[] = {{static_cast<const float*>(operand.first), hidden, width, ld, row_top, column_top, gate},
                           {static_cast<const float*>(operand.second), hidden, width, ld, second_row_top, column_top, up}};
  operand.first = gate; operand.second = up;
  operand.ld = ld; operand.part = hidden * ld;
  return launch_split(jobs, 2, stream);
}

// Widest matrices: a tile's offsets, up to 64 rows of 2 padded hidden values, fit 32 bits.
constexpr int64_t kMostColumns = int64_t{1} << 20;

constexpr TileSize kSizes[] = {kLarge, kMiddle, kSmall};
struct Shape {
  int64_t m, n;
  int64_t tiles_m(int64_t rows) const { return ceil_div(rows, m); }
  int64_t tiles_n(int64_t columns) const { return ceil_div(columns, n); }
};
template <typename Format>
Shape shape_of(TileSize size) {
  typedef Tiles<Format> All;
  if (size == kLarge) return {All::Large::kM, All::Large::kN};
  if (size == kMiddle) return {All::Middle::kM, All::Middle::kN};
  return {All::Small::kM, All::Small::kN};
}

// A product's tile size and how many runs its depth is cut into, by an estimate of its time. A tile
// size's workgroups run `resident` to a CU, together reach `rate` (TFLOP/s) and take `round` us beside
// it for their first loads and last stores; one alone on its CU takes `alone` of the time it takes
// among others. What the estimate decides is how the last, partly filled round weighs against the
// lower rates of smaller tiles, and, where a depth may be cut, against the partial results' bytes.
// The float32 figures are fitted. Over 1,486 measured products of 18 layers (64 to 65,536 rows, 128 to 4,096
// wide, 93 to 10,240 hidden) they give the time to 19 % rms, and what the plan takes is 0.6 % from the fastest
// tile and runs in the geometric mean and 7 % at most. The bfloat16 figures are large products' rates with one
// common round: over 742 products of these layers 29 % rms, and 8 % from the fastest, 92 % at most.
struct TileRate {
  int resident;
  double rate, alone, round;
};
template <typename Format>
TileRate tile_rate(TileSize size, bool direct, int64_t rows) {
  if (std::is_same_v<Format, HalfParts>) {
    if (size == kLarge) return split_before(size, rows) ? TileRate{1, 486, 1, 13.7} : TileRate{1, 299, 1, 12.7};
    return size == kMiddle ? TileRate{2, 202, 0.5, 18} : TileRate{4, 188, 0.77, 6.5};
  }
  if (std::is_same_v<Format, Bf16Parts>) {
    return size == kLarge ? TileRate{1, 248, 1, 17} : size == kMiddle ? TileRate{2, 179, 0.74, 6.3} : TileRate{4, 113, 0.8, 2.6};
  }
  if (direct) {
    return size == kLarge ? TileRate{1, 1250, 1, 3} : size == kMiddle ? TileRate{2, 1030, 0.6, 3} : TileRate{5, 470, 0.3, 3};
  }
  return size == kLarge ? TileRate{1, 1050, 1, 3} : size == kMiddle ? TileRate{2, 780, 0.6, 3} : TileRate{5, 410, 0.3, 3};
}

struct ProductPlan {
  TileSize size;
  int64_t runs;
  double us;
};

constexpr int64_t kMostRuns = 64;
template <typename Format>
ProductPlan product_plan(int64_t m, int64_t n, int64_t depth, bool direct, int64_t most_runs) {
  constexpr int64_t kShortest = 256;        // depth of a run
  constexpr double kBytesPerUs = 4e6, kJoinUs = 5.0;
  ProductPlan best{kSmall, 1, 1e30};
  for (TileSize size : kSizes) {
    const Shape shape = shape_of<Format>(size);
    const int64_t tiles = shape.tiles_m(m) * shape.tiles_n(n);
    const TileRate rate = tile_rate<Format>(size, direct, m);
    const int64_t slots = static_cast<int64_t>(kCus) * rate.resident;
    const int64_t longest = std::min(most_runs, std::max<int64_t>(depth / kShortest, 1));
    for (int64_t runs = 1; runs <= longest; ++runs) {
      const double full = 2.0 * shape.m * shape.n * (static_cast<double>(depth) / runs) * rate.resident / (rate.rate * 1e6 / kCus);
      const int64_t groups = tiles * runs, rest = groups % slots;
      double us = static_cast<double>(groups / slots) * (full + rate.round);
      if (rest > 0) {
        const double crowd = rate.resident == 1 ? 0 : static_cast<double>(ceil_div(rest, kCus) - 1) / (rate.resident - 1);
        us += full * (rate.alone + (1 - rate.alone) * crowd) + rate.round;
      }
      if (runs > 1) us += kJoinUs + 8.0 * runs * m * n / kBytesPerUs;
      if (us < best.us) best = {size, runs, us};
    }
  }
  return best;
}

// Whether x's and the weights' rows are whole, aligned 16 bytes of bfloat16.
bool whole_rows(const void* x, const void* gate_weight, const void* up_weight, int64_t width) {
  return width % 8 == 0 && aligned16(x) && aligned16(gate_weight) && aligned16(up_weight);
}

// What HalfParts takes beside its products: finding the scales (launches, the operands' bytes, and in
// the backward the maxima in the gate kernel, whose atomics grow with the rows) and, for operands split
// before, their parts (4,000 x 256 x 683 training: 128 us with HalfParts; 30,000 x 200 x 200 241, and
// 226 with Bf16Parts; 8,000 x 150 x 2,000 330 and 408).
constexpr double kForwardTopsUs = 10.0, kBackwardTopsUs = 18.0, kRowTopUs = 4e-4;
double tops_us(int64_t values) { return 4.0 * static_cast<double>(values) / 4e6; }
double split_us(bool split, int64_t values) { return split ? 5.0 + 8.0 * static_cast<double>(values) / 4e6 : 0.0; }
// Narrower layers are outside what the estimates were fitted to.
constexpr int64_t kHalvesWidth = 64;

// The workgroups of gated_short_kernel, which takes the float32 layers that leave it one a CU at most.
int64_t short_groups(int64_t rows, int64_t hidden) { return ceil_div(rows, kShortSide) * ceil_div(hidden, kShortSide); }

// Whether a float32 forward takes HalfParts: where its products, with the pass over x and the weights,
// are estimated shorter.
bool forward_halves(int64_t rows, int64_t width, int64_t hidden) {
  if (rows <= kFewRows || width < kHalvesWidth || short_groups(rows, hidden) <= kCus) return false;
  const ProductPlan halves = product_plan<HalfParts>(rows, 2 * hidden, width, false, 1);
  return halves.us + kForwardTopsUs + tops_us((rows + 2 * hidden) * width) +
             split_us(split_before(halves.size, rows), 2 * hidden * width) <
         product_plan<Bf16Parts>(rows, 2 * hidden, width, false, 1).us;
}

size_t forward_tops_bytes(int64_t rows, int64_t hidden) { return align256(static_cast<size_t>(rows + 2 * hidden) * sizeof(unsigned)); }

struct BackwardPlan {
  int64_t pitch, sum_groups;
  ProductPlan dx, dw;
  bool halves;
  size_t gates, sums, partials, tops, parts, total;  // offsets of the buffers
};

template <typename Format>
void plan_products(BackwardPlan& p, int64_t rows, int64_t width, bool direct) {
  p.dx = product_plan<Format>(rows, width, 2 * p.pitch, direct, kMostRuns);
  p.dw = product_plan<Format>(2 * p.pitch, width, rows, direct, kMostRuns);
}

template <typename T>
BackwardPlan backward_plan(int64_t rows, int64_t width, int64_t hidden, bool direct) {
  BackwardPlan p;
  constexpr size_t size = sizeof(T);
  p.pitch = padded(hidden);
  p.sum_groups = std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, 16), std::max<int64_t>(1, 2048 / ceil_div(p.pitch, 256))));
  p.halves = false;
  if constexpr (std::is_same_v<T, float>) {
    plan_products<Bf16Parts>(p, rows, width, false);
    BackwardPlan halves = p;
    plan_products<HalfParts>(halves, rows, width, false);
    if (width >= kHalvesWidth &&
        halves.dx.us + halves.dw.us + kBackwardTopsUs + kRowTopUs * static_cast<double>(rows) +
                tops_us((rows + 2 * hidden) * width) +
                split_us(split_before(halves.dx.size, rows), 2 * hidden * width) +
                split_us(split_before(halves.dw.size, 2 * p.pitch), rows * width) <
            p.dx.us + p.dw.us) {
      p = halves;
      p.halves = true;
      // Every workgroup of the gate kernel ends with an atomic a column: few and long ones, two a CU.
      p.sum_groups = std::max<int64_t>(1, std::min(ceil_div(rows, 64), 2 * kCus / ceil_div(p.pitch, 256)));
    }
  } else {
    plan_products<Bf16>(p, rows, width, direct);
  }
  p.gates = 0;
  p.sums = align256(static_cast<size_t>(rows) * 2 * p.pitch * size);
  p.partials = p.sums + align256(static_cast<size_t>(p.sum_groups) * 2 * p.pitch * sizeof(float));
  size_t partial = 0;
  if (p.dx.runs > 1) partial = static_cast<size_t>(p.dx.runs) * rows * width * sizeof(float);
  if (p.dw.runs > 1) partial = std::max(partial, static_cast<size_t>(p.dw.runs) * 2 * p.pitch * width * sizeof(float));
  p.tops = p.partials + align256(partial);
  // dg and du by rows and by columns, the weights and x by columns.
  p.parts = p.tops + (p.halves ? align256(static_cast<size_t>(rows + 2 * p.pitch + 2 * width) * sizeof(unsigned)) : 0);
  // The weights' parts, and when their product is done x's.
  size_t parts = 0;
  if (p.halves && split_before(p.dx.size, rows)) parts = split_bytes(2 * hidden, width);
  if (p.halves && split_before(p.dw.size, 2 * p.pitch)) parts = std::max(parts, split_bytes(rows, width));
  p.total = p.parts + parts;
  return p;
}

template <typename Format, Source kSourceA, Source kSourceB>
int launch_product(ProductArgs args, ProductPlan plan, Staging staging, float* partials, hipStream_t stream) {
  const Shape shape = shape_of<Format>(plan.size);
  args.tiles_m = shape.tiles_m(args.rows);
  args.tiles_n = shape.tiles_n(args.columns);
  args.partials = plan.runs > 1 ? partials : nullptr;
  const auto go = [&](auto tile, auto how) {
    typedef decltype(tile) G;
    args.steps = ceil_div(args.a.depth, G::kDepth);
    const dim3 grid(static_cast<unsigned>(args.tiles_m * args.tiles_n), static_cast<unsigned>(plan.runs));
    product_kernel<G, decltype(how)::value, kSourceA, kSourceB><<<grid, G::kThreads, 0, stream>>>(args);
  };
  if (plan.size == kLarge) with_staging<Format, typename Tiles<Format>::Large>(staging, go);
  else if (plan.size == kMiddle) with_staging<Format, typename Tiles<Format>::Middle>(staging, go);
  else with_staging<Format, typename Tiles<Format>::Small>(staging, go);
  if (int status = check_launch("gated linear product")) return status;
  if (plan.runs > 1) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(args.rows * ceil_div(args.columns, 4), 256), 4096));
    join_kernel<typename Format::T><<<grid, 256, 0, stream>>>(args, static_cast<int>(plan.runs));
    return check_launch("gated linear join");
  }
  return FHOAD_SUCCESS;
}

int check_sizes(int64_t rows, int64_t width, int64_t hidden, int activation, int dtype) {
  if (int status = check_dtype(dtype)) return status;
  if (activation < FHOAD_SILU || activation > FHOAD_SIGMOID) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "unknown activation %d", activation);
  }
  constexpr int64_t kMost = int64_t{1} << 31;
  if (rows < 0 || rows >= kMost || width < 1 || width > kMostColumns || hidden < 1 || hidden > kMostColumns) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "rows must be 0 to 2^31 - 1, width and hidden 1 to 2^20");
  }
  if (ceil_div(rows, 64) * ceil_div(2 * padded(hidden), 64) >= kMost ||
      ceil_div(rows, 64) * ceil_div(width, 64) >= kMost ||
      ceil_div(2 * padded(hidden), 64) * ceil_div(width, 64) >= kMost) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "the product has too many tiles");
  }
  return FHOAD_SUCCESS;
}

template <typename Format>
int launch_forward(ForwardArgs args, TileSize size, Staging staging, hipStream_t stream) {
  const Shape shape = shape_of<Format>(size);
  args.tiles_m = shape.tiles_m(args.rows);
  args.tiles_n = shape.tiles_n(2 * args.hidden);
  const auto go = [&](auto tile, auto how) {
    typedef decltype(tile) G;
    gated_forward_kernel<G, decltype(how)::value><<<static_cast<unsigned>(args.tiles_m * args.tiles_n), G::kThreads, 0, stream>>>(args);
  };
  if (size == kLarge) with_staging<Format, typename Tiles<Format>::Large>(staging, go);
  else if (size == kMiddle) with_staging<Format, typename Tiles<Format>::Middle>(staging, go);
  else with_staging<Format, typename Tiles<Format>::Small>(staging, go);
  return check_launch("gated linear forward");
}

template <typename T>
int forward(const void* x, const void* gate_weight, const void* up_weight, const void* gate_bias,
            const void* up_bias, void* h, float* pre, void* workspace, int64_t rows, int64_t width,
            int64_t hidden, int activation, hipStream_t stream) {
  ForwardArgs args{};
  args.x = {x, nullptr, width, rows, width, 0, 0, nullptr, nullptr};
  args.weights = {gate_weight, up_weight, width, hidden, width, 0, 0, nullptr, nullptr};
  args.gate_bias = gate_bias; args.up_bias = up_bias; args.h = h; args.pre = pre;
  args.rows = rows; args.hidden = hidden; args.pre_pitch = padded(hidden);
  args.activation = activation;
  if (rows <= kFewRows) {
    const auto go = [&](auto blocks) {
      constexpr int kBlocks = decltype(blocks)::value;
      constexpr bool kFloat = std::is_same_v<T, float>;
      if (hidden >= 4096) {  // enough features for every CU without more waves
        constexpr int kPairs = kFloat ? 2 : 1, kWaves = kFloat ? 8 : 4;
        gated_few_rows_kernel<T, kBlocks, kPairs, kWaves>
            <<<static_cast<unsigned>(ceil_div(hidden, 16 * kPairs)), kWaves * kWave, 0, stream>>>(args);
      } else {
        gated_few_rows_kernel<T, kBlocks, 1, 8><<<static_cast<unsigned>(ceil_div(hidden, 16)), 8 * kWave, 0, stream>>>(args);
      }
    };
    rows <= 16 ? go(std::integral_constant<int, 1>()) : go(std::integral_constant<int, 2>());
    return check_launch("gated linear forward");
  }
  if constexpr (std::is_same_v<T, float>) {
    if (short_groups(rows, hidden) <= kCus) {
      const dim3 grid(static_cast<unsigned>(ceil_div(hidden, kShortSide)), static_cast<unsigned>(ceil_div(rows, kShortSide)));
      gated_short_kernel<<<grid, kShortWaves * kWave, 0, stream>>>(args);
      return check_launch("gated linear forward");
    }
    if (!forward_halves(rows, width, hidden)) {
      return launch_forward<Bf16Parts>(args, product_plan<Bf16Parts>(rows, 2 * hidden, width, false, 1).size, kRegisters, stream);
    }
    unsigned* const tops = static_cast<unsigned*>(workspace);
    const TopJob jobs[] = {{static_cast<const float*>(x), rows, width, tops, nullptr},
                           {static_cast<const float*>(gate_weight), hidden, width, tops + rows, nullptr},
                           {static_cast<const float*>(up_weight), hidden, width, tops + rows + hidden, nullptr}};
    if (int status = launch_tops(tops, rows + 2 * hidden, jobs, 3, stream)) return status;
    args.x.top = tops;
    args.weights.top = tops + rows;
    args.weights.second_top = tops + rows + hidden;
    const TileSize size = product_plan<HalfParts>(rows, 2 * hidden, width, false, 1).size;
    const bool split = split_before(size, rows);
    if (split) {
      char* const parts = static_cast<char*>(workspace) + forward_tops_bytes(rows, hidden);
      if (int status = split_weights(args.weights, hidden, width, args.weights.top, args.weights.second_top, nullptr, parts, stream)) {
        return status;
      }
    }
    return launch_forward<HalfParts>(args, size, split ? kPlanes : kRegisters, stream);
  } else {
    const bool direct = whole_rows(x, gate_weight, up_weight, width);
    return launch_forward<Bf16>(args, product_plan<Bf16>(rows, 2 * hidden, width, direct, 1).size, direct ? kDirect : kRegisters, stream);
  }
}

template <typename T, typename Run>
int with_format(bool halves, Run run) {
  if constexpr (std::is_same_v<T, float>) return halves ? run(HalfParts{}) : run(Bf16Parts{});
  else return run(Bf16{});
}

template <typename T>
int backward(const void* x, const void* gate_weight, const void* up_weight, const float* pre,
             const void* grad_h, void* grad_x, void* grad_gate_weight, void* grad_up_weight,
             void* grad_gate_bias, void* grad_up_bias, void* workspace, int64_t rows, int64_t width,
             int64_t hidden, int activation, int dtype, hipStream_t stream) {
  const bool direct = whole_rows(x, gate_weight, up_weight, width);
  const BackwardPlan plan = backward_plan<T>(rows, width, hidden, direct);
  const Staging staging = direct && std::is_same_v<T, __bf16> ? kDirect : kRegisters;
  char* const base = static_cast<char*>(workspace);
  float* const sums = reinterpret_cast<float*>(base + plan.sums);
  float* const partials = reinterpret_cast<float*>(base + plan.partials);
  GateArgs gate{};
  gate.grad_h = grad_h; gate.pre = pre; gate.out = base + plan.gates;
  gate.partials = grad_gate_bias || grad_up_bias ? sums : nullptr;
  gate.rows = rows; gate.hidden = hidden; gate.pitch = plan.pitch;
  gate.rows_each = ceil_div(rows, plan.sum_groups);
  gate.activation = activation;
  // The scales' arrays: dg and du by rows, by columns, the weights by columns, x by columns.
  unsigned* const tops = reinterpret_cast<unsigned*>(base + plan.tops);
  unsigned *const column_top = tops + rows, *const weight_top = column_top + 2 * plan.pitch, *const x_top = weight_top + width;
  const dim3 gate_grid(static_cast<unsigned>(ceil_div(plan.pitch, 256)), static_cast<unsigned>(plan.sum_groups));
  if constexpr (std::is_same_v<T, float>) {
    if (plan.halves) {
      const TopJob jobs[] = {{static_cast<const float*>(gate_weight), hidden, width, nullptr, weight_top},
                             {static_cast<const float*>(up_weight), hidden, width, nullptr, weight_top},
                             {static_cast<const float*>(x), rows, width, nullptr, x_top}};
      if (int status = launch_tops(tops, rows + 2 * plan.pitch + 2 * width, jobs, 3, stream)) return status;
      gate.row_top = tops;
      gate.column_top = column_top;
      gate_backward_kernel<T, true><<<gate_grid, kGateWaves<true> * kWave, 0, stream>>>(gate);
    } else {
      gate_backward_kernel<T, false><<<gate_grid, kGateWaves<false> * kWave, 0, stream>>>(gate);
    }
  } else {
    gate_backward_kernel<T, false><<<gate_grid, kGateWaves<false> * kWave, 0, stream>>>(gate);
  }
  if (int status = check_launch("gate backward")) return status;
  const ColumnSum jobs[] = {{sums, grad_gate_bias, plan.sum_groups, 2 * plan.pitch, 0, 1},
                            {sums + plan.pitch, grad_up_bias, plan.sum_groups, 2 * plan.pitch, 0, 1}};
  if (int status = launch_column_sums(jobs, 2, hidden, dtype, stream)) return status;
  if (grad_x) {
    ProductArgs args{};
    args.a = {gate.out, nullptr, 2 * plan.pitch, rows, 2 * plan.pitch, 0, 0, tops, nullptr};
    args.b = {gate_weight, up_weight, width, width, 2 * plan.pitch, plan.pitch, hidden, weight_top, nullptr};
    args.first = grad_x;
    args.rows = args.half = args.segment = rows;
    args.columns = width;
    const bool split = plan.halves && split_before(plan.dx.size, rows);
    if (split) {
      if (int status = split_weights(args.b, hidden, width, nullptr, nullptr, weight_top, base + plan.parts, stream)) {
        return status;
      }
    }
    const auto run = [&](auto format) {
      return launch_product<decltype(format), kRows, kPairedColumns>(args, plan.dx, split ? kPlanes : staging, partials, stream);
    };
    if (int status = with_format<T>(plan.halves, run)) return status;
  }
  if (grad_gate_weight) {
    ProductArgs args{};
    args.a = {gate.out, nullptr, 2 * plan.pitch, 2 * plan.pitch, rows, 0, 0, column_top, nullptr};
    args.b = {x, nullptr, width, width, rows, 0, 0, x_top, nullptr};
    args.first = grad_gate_weight; args.second = grad_up_weight;
    args.rows = 2 * plan.pitch; args.half = plan.pitch; args.segment = hidden;
    args.columns = width;
    const bool split = plan.halves && split_before(plan.dw.size, 2 * plan.pitch);
    if (split) {
      const int64_t ld = split_ld(width);
      const SplitJob job{static_cast<const float*>(x), rows, width, ld, nullptr, x_top, reinterpret_cast<_Float16*>(base + plan.parts)};
      if (int status = launch_split(&job, 1, stream)) return status;
      args.b.first = job.out;
      args.b.ld = ld;
      args.b.part = rows * ld;
    }
    const auto run = [&](auto format) {
      return launch_product<decltype(format), kColumns, kColumns>(args, plan.dw, split ? kPlanes : staging, partials, stream);
    };
    return with_format<T>(plan.halves, run);
  }
  return FHOAD_SUCCESS;
}

}  // namespace
}  // namespace fhoad_net

using namespace fhoad_net;

extern "C" size_t fhoad_gated_linear_saved_size(int64_t rows, int64_t hidden) {
  return rows <= 0 || hidden <= 0 ? 0 : static_cast<size_t>(rows) * 2 * padded(hidden) * sizeof(float);
}

extern "C" size_t fhoad_gated_linear_forward_workspace_size(int64_t rows, int64_t width, int64_t hidden, int dtype) {
  if (dtype != FHOAD_FLOAT32 || rows <= 0 || width <= 0 || hidden <= 0 || !forward_halves(rows, width, hidden)) return 0;
  const bool split = split_before(product_plan<HalfParts>(rows, 2 * hidden, width, false, 1).size, rows);
  return forward_tops_bytes(rows, hidden) + (split ? split_bytes(2 * hidden, width) : 0);
}

extern "C" int fhoad_gated_linear_forward(const void* x, const void* gate_weight, const void* up_weight,
                                          const void* gate_bias, const void* up_bias, void* h, float* pre,
                                          void* workspace, size_t workspace_bytes, int64_t rows, int64_t width,
                                          int64_t hidden, int activation, int dtype, void* stream) {
  if (int status = check_sizes(rows, width, hidden, activation, dtype)) return status;
  if (rows == 0) return FHOAD_SUCCESS;
  if (!x || !gate_weight || !up_weight || !h) return fail(FHOAD_ERROR_INVALID_VALUE, "null device pointer");
  if (!aligned16(pre)) return fail(FHOAD_ERROR_MISALIGNED, "pre must be 16-byte aligned");
  if (int status = check_workspace(workspace, workspace_bytes,
                                   fhoad_gated_linear_forward_workspace_size(rows, width, hidden, dtype))) {
    return status;
  }
  const auto run = dtype == FHOAD_FLOAT32 ? forward<float> : forward<__bf16>;
  return run(x, gate_weight, up_weight, gate_bias, up_bias, h, pre, workspace, rows, width, hidden, activation,
             static_cast<hipStream_t>(stream));
}

extern "C" size_t fhoad_gated_linear_backward_workspace_size(int64_t rows, int64_t width, int64_t hidden,
                                                             int dtype) {
  if (rows <= 0 || width <= 0 || hidden <= 0) return 0;
  // Pointers decide between the two ways of staging, and so do plans: enough for both.
  if (dtype == FHOAD_FLOAT32) return backward_plan<float>(rows, width, hidden, false).total;
  return std::max(backward_plan<__bf16>(rows, width, hidden, false).total,
                  backward_plan<__bf16>(rows, width, hidden, true).total);
}

extern "C" int fhoad_gated_linear_backward(const void* x, const void* gate_weight, const void* up_weight,
                                           const float* pre, const void* grad_h, void* grad_x,
                                           void* grad_gate_weight, void* grad_up_weight,
                                           void* grad_gate_bias, void* grad_up_bias, void* workspace,
                                           size_t workspace_bytes, int64_t rows, int64_t width,
                                           int64_t hidden, int activation, int dtype, void* stream) {
  if (int status = check_sizes(rows, width, hidden, activation, dtype)) return status;
  if (!grad_gate_weight != !grad_up_weight) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "the weights' gradients come together");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows == 0) {
    for (void* weight : {grad_gate_weight, grad_up_weight}) {
      if (int status = zero(weight, hidden * width, dtype, s)) return status;
    }
    for (void* bias : {grad_gate_bias, grad_up_bias}) {
      if (int status = zero(bias, hidden, dtype, s)) return status;
    }
    return FHOAD_SUCCESS;
  }
  if (!x || !gate_weight || !up_weight || !pre || !grad_h) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "null device pointer");
  }
  if (!aligned16(pre)) return fail(FHOAD_ERROR_MISALIGNED, "pre must be 16-byte aligned");
  if (int status = check_workspace(workspace, workspace_bytes,
                                   fhoad_gated_linear_backward_workspace_size(rows, width, hidden, dtype))) {
    return status;
  }
  const auto run = dtype == FHOAD_FLOAT32 ? backward<float> : backward<__bf16>;
  return run(x, gate_weight, up_weight, pre, grad_h, grad_x, grad_gate_weight, grad_up_weight, grad_gate_bias,
             grad_up_bias, workspace, rows, width, hidden, activation, dtype, s);
}
