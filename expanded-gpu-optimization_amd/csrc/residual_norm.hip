// Residual, gate and norms between two blocks (fhoad_residual_norm_forward / _backward).
//
// With n = norm(block) or block, the forward is hidden = scale residual + gate n and
// normed = norm(hidden). The backward, with t the gradient of hidden's sum of uses:
//   xhat = (hidden - mean) rstd,  d = grad_normed weight
//   t = grad_hidden + rstd (d - xhat mean(d xhat) - mean(d))        (the last term: layer norm)
//   grad_residual = scale t,  grad_gate = sum of t n,  dn = t gate
//   grad_block = the same form as t's second term, of dn through the first norm
// and the weights' gradients are sums over the rows. The forward moves 4 values an element (residual,
// block in; hidden, normed out), the backward 6, and some 40 float operations each way stay far below
// the memory's time.
//
// A row is held in registers by one wave (up to 512 or 1,024 values) or by one workgroup, so the two
// norms need no second read; only the backward of rows above 8,192 columns reads a row again in each of
// its passes, from the caches. The backward forms hidden again from residual and block: the same
// bytes as reading it, and with bfloat16 without its rounding. Column sums stay with their threads over
// all rows of a workgroup, in registers (above 4,096 columns some of them in LDS), and meet in a second,
// small launch in a fixed order.
#include "network_common.h"

#include <algorithm>
#include <type_traits>

namespace fhoad_net {
namespace {

struct NormArgs {
  const void *residual, *block, *gate, *weight, *bias, *post_weight, *post_bias;
  const void *grad_hidden, *grad_normed;
  void *hidden, *normed, *grad_residual, *grad_block, *grad_gate;
  float* statistics;  // [rows][4]: post mean, post rstd, mean, rstd
  float* partials;    // backward: [workgroups][4][width], then gate partials [units][width]
  int64_t rows, width, rows_per_gate;
  // Work of the backward: `units` runs of `unit_rows` rows, `splits` of them to a gate row.
  int64_t units, splits, unit_rows;
  float scale, eps;
  int layer;
  int element_gate;
  int want_sums;  // weights', biases' gradients
};

// How a row lies over its threads: 16-byte vector j of thread t starts at element
// (j kThreads + t) kVec. kWhole: rows are whole, aligned vectors. Otherwise vectors are read and
// written at their elements' alignment, which the hardware allows at full speed, and a row's last
// vector is read from kVec before the row's end: its first elements are the vector's before, not
// `inside` (read element by element, that one vector held up each row: 1,365 bfloat16 took three times
// as long).
template <typename T_, int kPer_, int kThreads_, bool kWhole>
struct Row {
  typedef T_ T;
  static constexpr int kPer = kPer_, kThreads = kThreads_;
  static constexpr int kVec = 16 / static_cast<int>(sizeof(T)), kVectors = kPer / kVec;
  typedef T V __attribute__((ext_vector_type(kVec)));
  struct __attribute__((packed, aligned(alignof(T)))) Loose {
    V v;
  };

  static __device__ __forceinline__ int first(int j, int t) { return (j * kThreads + t) * kVec; }
  // Where vector j of thread t is read.
  static __device__ __forceinline__ int start(int j, int t, int width) {
    return kWhole ? first(j, t) : min(first(j, t), width - kVec);
  }
  // The column of element e of thread t.
  static __device__ __forceinline__ int column(int e, int t, int width) { return start(e / kVec, t, width) + e % kVec; }
  // Whether it is the row's (and no other vector's).
  static __device__ __forceinline__ bool inside(int e, int t, int width) {
    if constexpr (kWhole) return first(e / kVec, t) < width;
    return e % kVec >= first(e / kVec, t) - start(e / kVec, t, width);
  }
  // A row's address is the same for a wave: 32 bits a lane beside it.
  static __device__ __forceinline__ unsigned offset(int j, int t, int width) {
    return static_cast<unsigned>(start(j, t, width)) * static_cast<unsigned>(sizeof(T));
  }
  static __device__ __forceinline__ void load(V& x, const void* base, int64_t row, int j, int t, int width) {
    const T* p = static_cast<const T*>(base) + row * width;
    x = V{};
    if (kWhole || width >= kVec) {  // the same for every row
      const char* const at = reinterpret_cast<const char*>(p) + offset(j, t, width);
      if (first(j, t) < width) x = kWhole ? *reinterpret_cast<const V*>(at) : reinterpret_cast<const Loose*>(at)->v;
    } else if (j == 0 && t == 0) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (i + width >= kVec) x[i] = p[i + width - kVec];
      }
    }
  }
  static __device__ __forceinline__ void load(V (&x)[kVectors], const void* base, int64_t row, int t,
                                              int width) {
#pragma unroll
    for (int j = 0; j < kVectors; ++j) load(x[j], base, row, j, t, width);
  }
  static __device__ __forceinline__ void store(void* base, int64_t row, int t, int width,
                                               const float (&x)[kPer]) {
    T* p = static_cast<T*>(base) + row * width;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      if (first(j, t) >= width) continue;
      V v;
#pragma unroll
      for (int i = 0; i < kVec; ++i) v[i] = from_float<T>(x[j * kVec + i]);
      char* const at = reinterpret_cast<char*>(p) + offset(j, t, width);
      if constexpr (kWhole) {
        *reinterpret_cast<V*>(at) = v;
      } else if (first(j, t) + kVec <= width) {
        reinterpret_cast<Loose*>(at)->v = v;
      } else if (width >= kVec) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          if (inside(j * kVec + i, t, width)) reinterpret_cast<T*>(at)[i] = v[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          if (i + width >= kVec) p[i + width - kVec] = v[i];
        }
      }
    }
  }
};

// Sums of two values over a row's threads. With one wave to a row nothing is shared; otherwise
// the waves meet in LDS, in two buffers by turns, so that one barrier is enough: a buffer is
// written again only after the next meeting's barrier, which every reader of it has passed.
template <int kThreads>
struct RowSums {
  float (*shared)[2][16];
  int turn = 0;

  __device__ __forceinline__ f2 operator()(float a, float b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (kThreads > kWave) {
      const int wave = threadIdx.x / kWave;
      if (threadIdx.x % kWave == 0) {
        shared[turn][0][wave] = a;
        shared[turn][1][wave] = b;
      }
      __syncthreads();
      a = b = 0.0f;
#pragma unroll
      for (int w = 0; w < kThreads / kWave; ++w) {
        a += shared[turn][0][w];
        b += shared[turn][1][w];
      }
      turn ^= 1;
    }
    return f2{a, b};
  }
};

// The thread's place, as if it were new in each row: with rows that are not whole, the compiler would
// otherwise form every element's `inside` before the loop, 16 scalar registers too many for each 8.
template <bool kWhole>
__device__ __forceinline__ int anew(int t) {
  if constexpr (!kWhole) asm volatile("" : "+v"(t));
  return t;
}

template <int kThreads>
constexpr int kGroup = kThreads == kWave ? 256 : kThreads;  // workgroup size
template <int kThreads>
constexpr int kRowsAtOnce = kGroup<kThreads> / kThreads;
// Which of a workgroup's rows a thread is at, the same for its wave.
template <int kThreads>
__device__ __forceinline__ int row_group() {
  return kRowsAtOnce<kThreads> == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
}

// Mean (layer norm) and 1 / sqrt(mean of squares + eps) of a row: the mean is taken out before
// the squares are summed, so a large common offset costs no precision.
template <typename R, typename Get>
__device__ __forceinline__ f2 row_statistics(RowSums<R::kThreads>& sums, int t, int width, int layer,
                                             float eps, Get get) {
  constexpr int kPer = R::kPer;
  const float inverse = 1.0f / static_cast<float>(width);
  float mean = 0.0f;
  if (layer) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum += R::inside(e, t, width) ? get(e) : 0.0f;
    mean = sums(sum, 0.0f)[0] * inverse;
  }
  float squares = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const float d = R::inside(e, t, width) ? get(e) - mean : 0.0f;
    squares += d * d;
  }
  const float square = sums(squares, 0.0f)[0] * inverse;
  return f2{mean, 1.0f / __builtin_sqrtf(square + eps)};
}

// Bound by memory: 65,536 x 256 float32 44 us (6.1 TB/s of 268 MB, part of it from the cache), 16,384 x
// 4,096 bfloat16 106 us (5.1 TB/s), 5,003 x 1,365 float32 with an element's gate and rows at any alignment
// 30 us (4.6 TB/s). A workgroup's rows are consecutive, so a gate's row and the
// weights are read once.
template <typename T, int kPer, int kThreads, bool kWhole>
__global__ __launch_bounds__(kGroup<kThreads>) void norm_forward_kernel(NormArgs a) {
  typedef Row<T, kPer, kThreads, kWhole> R;
  typedef typename R::V V;
  constexpr int kVectors = R::kVectors, kVec = R::kVec;
  __shared__ float s_sums[2][2][16];
  RowSums<kThreads> sums{s_sums};
  const int width = static_cast<int>(a.width);
  const int thread = threadIdx.x % kThreads;
  const int64_t per = ceil_div(a.rows, static_cast<int64_t>(gridDim.x) * kRowsAtOnce<kThreads>);
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kRowsAtOnce<kThreads> + row_group<kThreads>()) * per;
  const int64_t last = min(first + per, a.rows);

  V weight[kVectors], bias[kVectors], post_weight[kVectors], post_bias[kVectors], gate[kVectors];
  R::load(weight, a.weight, 0, thread, width);
  if (a.bias) R::load(bias, a.bias, 0, thread, width);
  if (a.post_weight) R::load(post_weight, a.post_weight, 0, thread, width);
  if (a.post_bias) R::load(post_bias, a.post_bias, 0, thread, width);
  int64_t gate_row = -1;
  for (int64_t row = first; row < last; ++row) {
    const int t = anew<kWhole>(thread);
    V x[kVectors], y[kVectors];
    R::load(x, a.residual, row, t, width);
    if (a.block) R::load(y, a.block, row, t, width);
    if (a.gate) {
      const int64_t wanted = row / a.rows_per_gate;
      if (wanted != gate_row) R::load(gate, a.gate, wanted, t, width);
      gate_row = wanted;
    }
    f2 post = {0.0f, 0.0f};
    float h[kPer];
    if (a.post_weight) {
      post = row_statistics<R>(sums, t, width, a.layer, a.eps, [&](int e) {
        return to_float(y[e / kVec][e % kVec]);
      });
    }
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        float v = a.scale * to_float(x[j][i]);
        if (a.block) {
          float n = to_float(y[j][i]);
          if (a.post_weight) {
            n = (n - post[0]) * post[1] * to_float(post_weight[j][i]);
            if (a.post_bias) n += to_float(post_bias[j][i]);
          }
          v += a.gate ? to_float(gate[j][i]) * n : n;
        }
        h[j * kVec + i] = R::inside(j * kVec + i, t, width) ? v : 0.0f;
      }
    }
    if (a.hidden) R::store(a.hidden, row, t, width, h);
    const f2 own = row_statistics<R>(sums, t, width, a.layer, a.eps,
                                                           [&](int e) { return h[e]; });
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        float v = (h[j * kVec + i] - own[0]) * own[1] * to_float(weight[j][i]);
        if (a.bias) v += to_float(bias[j][i]);
        h[j * kVec + i] = v;
      }
    }
    R::store(a.normed, row, t, width, h);
    if (a.statistics && t == 0) {
      *reinterpret_cast<f4*>(a.statistics + 4 * row) = f4{post[0], post[1], own[0], own[1]};
    }
  }
}

// Adds a workgroup's column sums (its rows' groups of 64 threads meet in LDS, in order) and writes
// them as a row of `out`, as T. Every thread of the workgroup calls this.
template <typename R, typename Out>
__device__ __forceinline__ void write_sums(float* s_row, Out* out, int width, const float (&sum)[R::kPer]) {
  constexpr int kThreads = R::kThreads, kPer = R::kPer;
  const int t = threadIdx.x % kThreads;
  if constexpr (kRowsAtOnce<kThreads> == 1) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (R::inside(e, t, width)) out[R::column(e, t, width)] = from_float<Out>(sum[e]);
    }
  } else {
    const int group = threadIdx.x / kThreads;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (R::inside(e, t, width)) s_row[group * (kPer * kThreads) + R::column(e, t, width)] = sum[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += kGroup<kThreads>) {
      float total = 0.0f;
#pragma unroll
      for (int g = 0; g < kRowsAtOnce<kThreads>; ++g) total += s_row[g * (kPer * kThreads) + c];
      out[c] = from_float<Out>(total);
    }
  }
}

// A column sum over a workgroup's rows, kPer values of each thread, in registers or in LDS.
template <int kPer, int kThreads, bool kInLds>
struct ColumnTotal {
  f4 value[kInLds ? 1 : kPer / 4];
  f4* lds;

  __device__ __forceinline__ explicit ColumnTotal(f4* shared) : lds(shared + threadIdx.x % kThreads) { clear(); }
  __device__ __forceinline__ f4& at(int quad) { return kInLds ? lds[quad * kThreads] : value[kInLds ? 0 : quad]; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int q = 0; q < kPer / 4; ++q) at(q) = f4{};
  }
  __device__ __forceinline__ void get(float (&sum)[kPer]) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum[e] = at(e / 4)[e % 4];
  }
};

// What the backward reads of a row.
template <typename R, bool kElementGate>
struct BackwardRow {
  typename R::V x[R::kVectors], y[R::kVectors], dh[R::kVectors], dy[R::kVectors];
  typename R::V gate[kElementGate ? R::kVectors : 1];
  f4 statistics;

  __device__ __forceinline__ void load(const NormArgs& a, int64_t row, int t, int width) {
    R::load(x, a.residual, row, t, width);
    if (a.block) R::load(y, a.block, row, t, width);
    if (a.grad_hidden) R::load(dh, a.grad_hidden, row, t, width);
    if (a.grad_normed) R::load(dy, a.grad_normed, row, t, width);
    if constexpr (kElementGate) R::load(gate, a.gate, row, t, width);
    statistics = *reinterpret_cast<const f4*>(a.statistics + 4 * row);
  }
};

// Waves a SIMD that the backward is held to. Rows of bfloat16 that are not whole vectors, without a norm
// after the block, need a few registers more or less than the 128 of four waves: held to four, 500, 1,365
// and 3,001 columns take 169, 174 and 174 us (60 million values), left alone 178, 175 to 199 and 182. Whole
// rows are left alone: 4,096 columns 156 us, held to four 166.
template <typename T, int kThreads, bool kWhole, bool kPost>
constexpr int kBackwardWaves = sizeof(T) == 2 && !kWhole && !kPost && kThreads < 1024 ? 4 : 1;

// kPost: there is a norm after the block. kElementGate: a gate for each element, whose gradient is
// written with the row's; otherwise a gate shared by rows or none.
// Bound by memory: 65,536 x 256 float32 81 us (5.0 TB/s), 16,384 x 4,096 bfloat16 171 us (4.7 TB/s), 5,003 x
// 1,365 float32 with an element's gate 43 us (5.1 TB/s). Up to five column sums a value stay in registers,
// which leaves two or three waves a SIMD: too few to cover the loads without the next row's being under way
// (before that, and with one kernel for every kind of gate, 16,384 x 4,096 took 280 us).
template <typename T, int kPer, int kThreads, bool kWhole, bool kPost, bool kElementGate>
__global__ __launch_bounds__(kGroup<kThreads>, (kBackwardWaves<T, kThreads, kWhole, kPost>)) void norm_backward_kernel(NormArgs a) {
  typedef Row<T, kPer, kThreads, kWhole> R;
  typedef typename R::V V;
  constexpr int kVectors = R::kVectors, kVec = R::kVec;
  // A thread of 1,024 has 128 registers. There the column sums that fit lie in LDS (a thread's own, 16 bytes
  // at a time), the weights are read again for each row, from the caches, and the next row is not read
  // ahead. All in registers, which then spill, 7,324 x 8,192 took 783 us in float32 and 569 in bfloat16
  // (now 296 and 182: 4.9 and 4.0 TB/s); with the next row ahead 472 and 200.
  // Above 8,192 columns a thread has 16 values and three sums of each in registers. There, a row's vectors
  // are read one at a time in each of the passes over it, the later times from the caches, and only xhat and
  // the gradient stay between (kReread). 4,882 x 12,288 in us, with all of a row held and now: no norm after
  // the block, float32 622 and 317 (4.5 TB/s), bfloat16 297 and 176 (4.1); element's gate 1,245 and 546
  // (4.3), 505 and 360. With a norm after the block and a shared gate five sums still spill: 1,540 and 1,120
  // (1.3 TB/s), 858 and 850.
  constexpr bool kWide = kThreads == 1024;
  constexpr bool kReread = kWide && kPer == 16;
  constexpr int kLdsTotals = !kWide ? 0 : kPer == 8 ? 4 : 2;
  constexpr bool kPrefetch = !kWide;
  typedef ColumnTotal<kPer, kThreads, (kLdsTotals > 0)> Total0;
  typedef ColumnTotal<kPer, kThreads, (kLdsTotals > 1)> Total1;
  typedef ColumnTotal<kPer, kThreads, (kLdsTotals > 2)> Total2;
  typedef ColumnTotal<kPer, kThreads, (kLdsTotals > 3)> Total3;
  __shared__ f4 s_total[kLdsTotals ? kLdsTotals * kPer / 4 * kThreads : 1];
  constexpr int kTotal = kLdsTotals ? kPer / 4 * kThreads : 0;
  __shared__ float s_sums[2][2][16];
  __shared__ float s_row[kRowsAtOnce<kThreads> == 1 ? 1 : kPer * kGroup<kThreads>];
  RowSums<kThreads> sums{s_sums};
  const int width = static_cast<int>(a.width);
  const float inverse = 1.0f / static_cast<float>(width);
  const int thread = threadIdx.x % kThreads, group = row_group<kThreads>();
  const bool summed_gate = !kElementGate && a.grad_gate;

  constexpr int kPostVectors = kPost ? kVectors : 1;
  Total0 d_weight(s_total);
  Total1 d_post_weight(s_total + kTotal);
  Total2 d_gate(s_total + 2 * kTotal);
  Total3 d_post_bias(s_total + 3 * kTotal);
  ColumnTotal<kPer, kThreads, false> d_bias(nullptr);
  V weight[kVectors], post_weight[kPostVectors], post_bias[kPostVectors], shared_gate[kElementGate ? 1 : kVectors];
  const auto load_weights = [&](int64_t gate_row, int t) {
    R::load(weight, a.weight, 0, t, width);
    if constexpr (kPost) {
      R::load(post_weight, a.post_weight, 0, t, width);
      if (a.post_bias) R::load(post_bias, a.post_bias, 0, t, width);
    }
    if constexpr (!kElementGate) {
      if (a.gate) R::load(shared_gate, a.gate, gate_row, t, width);
    }
  };

  const int64_t unit_end = a.units * (static_cast<int64_t>(blockIdx.x) + 1) / gridDim.x;
  for (int64_t unit = a.units * blockIdx.x / gridDim.x; unit < unit_end; ++unit) {
    const int64_t gate_row = unit / a.splits;
    const int64_t span = kElementGate ? a.rows : a.rows_per_gate;
    const int64_t begin = gate_row * span + (unit % a.splits) * a.unit_rows;
    const int64_t end = min(begin + a.unit_rows, (gate_row + 1) * span);
    if constexpr (!kElementGate) d_gate.clear();
    if constexpr (!kWide) load_weights(gate_row, thread);
    // The next row's values are on their way while a row is worked on.
    BackwardRow<R, kElementGate> next;
    if (kPrefetch && begin + group < end) next.load(a, begin + group, thread, width);
    for (int64_t row = begin + group; row < end; row += kRowsAtOnce<kThreads>) {
      const int t = anew<kWhole>(thread);
      if constexpr (!kPrefetch && !kReread) next.load(a, row, t, width);
      if constexpr (kWide && !kReread) load_weights(gate_row, t);
      BackwardRow<R, kElementGate> now = next;
      if constexpr (kReread) now.statistics = *reinterpret_cast<const f4*>(a.statistics + 4 * row);
      // With kReread, vector j of what a pass over the row needs.
      const auto begin_vector = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        return anew<false>(thread);
      };
      // A value that is not read is zero, so that none is kept from the pass before.
      const auto reread_block = [&](int j, int at) {
        now.y[j] = V{};
        if (a.block) R::load(now.y[j], a.block, row, j, at, width);
        if constexpr (kPost) {
          post_weight[j] = post_bias[j] = V{};
          R::load(post_weight[j], a.post_weight, 0, j, at, width);
          if (a.post_bias) R::load(post_bias[j], a.post_bias, 0, j, at, width);
        }
        if constexpr (kElementGate) {
          now.gate[j] = V{};
          R::load(now.gate[j], a.gate, row, j, at, width);
        } else {
          shared_gate[j] = V{};
          if (a.gate) R::load(shared_gate[j], a.gate, gate_row, j, at, width);
        }
      };
      const auto &x = now.x, &y = now.y, &dh = now.dh, &dy = now.dy;
      if (kPrefetch && row + kRowsAtOnce<kThreads> < end) next.load(a, row + kRowsAtOnce<kThreads>, t, width);
      const f4 s = now.statistics;
      float unit_x[kPer], grad[kPer];
      float first = 0.0f, second = 0.0f;
      const auto post_unit = [&](int j, int i) { return (to_float(y[j][i]) - s[0]) * s[1]; };
      const auto branch = [&](int j, int i) {  // n
        if constexpr (!kPost) return to_float(y[j][i]);
        float n = post_unit(j, i) * to_float(post_weight[j][i]);
        if (a.post_bias) n += to_float(post_bias[j][i]);
        return n;
      };
      const auto gated = [&](int j, int i, float v) {
        if constexpr (kElementGate) return v * to_float(now.gate[j][i]);
        return a.gate ? v * to_float(shared_gate[j][i]) : v;
      };
      f4 part[2];  // four columns' share of two sums
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        if constexpr (kReread) {
          const int at = begin_vector();
          R::load(now.x[j], a.residual, row, j, at, width);
          now.dy[j] = V{};
          if (a.grad_normed) R::load(now.dy[j], a.grad_normed, row, j, at, width);
          R::load(weight[j], a.weight, 0, j, at, width);
          reread_block(j, at);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int e = j * kVec + i;
          float h = a.scale * to_float(x[j][i]);
          if (a.block) {
            h += gated(j, i, branch(j, i));
          }
          unit_x[e] = R::inside(e, t, width) ? (h - s[2]) * s[3] : 0.0f;
          const float up = a.grad_normed ? to_float(dy[j][i]) : 0.0f;
          part[0][e % 4] = up * unit_x[e];
          part[1][e % 4] = up;
          if (e % 4 == 3) {
            d_weight.at(e / 4) += part[0];
            d_bias.at(e / 4) += part[1];
          }
          // Selected after the product: a column that a row's last vector holds again counts for nothing,
          // with an infinite weight, too. Its column sums are not written.
          grad[e] = R::inside(e, t, width) ? up * to_float(weight[j][i]) : 0.0f;
          first += grad[e] * unit_x[e];
          second += grad[e];
        }
      }
      f2 total = sums(first, second);
      float along = total[0] * inverse, level = a.layer ? total[1] * inverse : 0.0f, rstd = s[3];
      // Without grad_normed nothing of the second norm counts, whatever its statistics: they may be
      // non-finite in a row that the loss leaves out. kClear: its terms are cleared here, otherwise not
      // selected below. 4,882 x 12,288 float32 and bfloat16 without a norm after the block, in us: cleared 317
      // and 176, selected 415 and 194; 7,324 x 8,192 with one: 401 and 226, 364 and 209.
      constexpr bool kClear = kReread && !kPost;
      if constexpr (kClear) {
        if (!a.grad_normed) {
          along = level = rstd = 0.0f;
#pragma unroll
          for (int e = 0; e < kPer; ++e) unit_x[e] = grad[e] = 0.0f;
        }
      }
      first = second = 0.0f;
      float out[kPer];
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        if constexpr (kReread) {
          const int at = begin_vector();
          now.dh[j] = V{};
          if (a.grad_hidden) R::load(now.dh[j], a.grad_hidden, row, j, at, width);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int e = j * kVec + i;
          float g = rstd * (grad[e] - unit_x[e] * along - level);
          if (!kClear && !a.grad_normed) g = 0.0f;
          if (a.grad_hidden) g += to_float(dh[j][i]);
          out[e] = a.scale * g;
          grad[e] = g;
        }
      }
      if (a.grad_residual) R::store(a.grad_residual, row, t, width, out);
      if (!a.block) continue;
      f4 post_part[2];
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        if constexpr (kReread) reread_block(j, begin_vector());
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int e = j * kVec + i;
          const float g = R::inside(e, t, width) ? grad[e] : 0.0f;
          out[e] = g * branch(j, i);
          if constexpr (!kElementGate) {
            part[0][e % 4] = out[e];
            if (e % 4 == 3) d_gate.at(e / 4) += part[0];
          }
          float dn = gated(j, i, g);
          if constexpr (kPost) {
            const float hat = post_unit(j, i);
            post_part[0][e % 4] = dn * hat;
            post_part[1][e % 4] = dn;
            if (e % 4 == 3) {
              d_post_weight.at(e / 4) += post_part[0];
              d_post_bias.at(e / 4) += post_part[1];
            }
            dn *= to_float(post_weight[j][i]);
            first += dn * hat;
            second += dn;
          }
          grad[e] = dn;
        }
      }
      if constexpr (kElementGate) {
        if (a.grad_gate) R::store(a.grad_gate, row, t, width, out);
      }
      if constexpr (kPost) {
        total = sums(first, second);
        const float post_along = total[0] * inverse, post_level = a.layer ? total[1] * inverse : 0.0f;
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
          if constexpr (kReread) R::load(now.y[j], a.block, row, j, begin_vector(), width);
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const int e = j * kVec + i;
            grad[e] = s[1] * (grad[e] - post_unit(j, i) * post_along - post_level);
          }
        }
      }
      if (a.grad_block) R::store(a.grad_block, row, t, width, grad);
    }
    if constexpr (!kElementGate) {
      if (!summed_gate) continue;
      float sum[kPer];
      d_gate.get(sum);
      if (a.splits == 1) {
        write_sums<R>(s_row, static_cast<T*>(a.grad_gate) + gate_row * width, width, sum);
      } else {
        write_sums<R>(s_row, a.partials + (4 * static_cast<int64_t>(gridDim.x) + unit) * width, width, sum);
      }
    }
  }
  if (!a.want_sums) return;
  float* const partials = a.partials + 4 * static_cast<int64_t>(blockIdx.x) * width;
  float sum[kPer];
  if (!a.grad_normed) {
    d_weight.clear();
    d_bias.clear();
  }
  d_weight.get(sum);
  write_sums<R>(s_row, partials, width, sum);
  d_bias.get(sum);
  write_sums<R>(s_row, partials + width, width, sum);
  if constexpr (kPost) {
    d_post_weight.get(sum);
    write_sums<R>(s_row, partials + 2 * width, width, sum);
    d_post_bias.get(sum);
    write_sums<R>(s_row, partials + 3 * width, width, sum);
  }
}

template <typename T>
__global__ void zero_kernel(T* out, int64_t n) {
  const int64_t k = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (k < n) out[k] = static_cast<T>(0.0f);
}

int zero(void* out, int64_t n, int dtype, hipStream_t stream) {
  if (!out || n == 0) return FHOAD_SUCCESS;
  const unsigned grid = static_cast<unsigned>(ceil_div(n, 256));
  if (dtype == FHOAD_FLOAT32) zero_kernel<<<grid, 256, 0, stream>>>(static_cast<float*>(out), n);
  else zero_kernel<<<grid, 256, 0, stream>>>(static_cast<__bf16*>(out), n);
  return check_launch("zero");
}

// The layout of a row by its width: one wave to a row as long as it holds 8 values a lane, then a
// workgroup that grows with the width. The forward has 16 values a thread from 1,024 on (5,000 to 8,192
// columns with 8 on 1,024 threads: within 5 % of it, 30 % slower at 8,192 bfloat16), the backward, which
// holds five column sums as well, 8 as long as 1,024 threads allow.
template <bool kForward, typename Launch>
void with_layout(int64_t width, Launch launch) {
#define FHOAD_LAYOUT(threads, per) \
  if (width <= threads * per) return launch(std::integral_constant<int, threads>(), std::integral_constant<int, per>())
  FHOAD_LAYOUT(64, 8);
  if constexpr (kForward) {
    FHOAD_LAYOUT(64, 16);
    FHOAD_LAYOUT(256, 8);
    FHOAD_LAYOUT(256, 16);
    FHOAD_LAYOUT(512, 16);
  } else {
    FHOAD_LAYOUT(128, 8);
    FHOAD_LAYOUT(256, 8);
    FHOAD_LAYOUT(512, 8);
    FHOAD_LAYOUT(1024, 8);
  }
  FHOAD_LAYOUT(1024, 16);
#undef FHOAD_LAYOUT
}
static_assert(1024 * 16 == FHOAD_NORM_MAX_WIDTH, "widest layout");

int forward_rows_at_once(int64_t width) { return width <= 1024 ? 4 : 1; }
int backward_rows_at_once(int64_t width) { return width <= 512 ? 4 : 1; }

// Rows to a backward workgroup: as many workgroups as run at once, each with its column sums.
struct BackwardPlan {
  int64_t groups, splits, units, unit_rows;
};
BackwardPlan backward_plan(int64_t rows, int64_t width, int64_t rows_per_gate) {
  const int64_t most = width <= 2048 ? 1024 : width <= 4096 ? 512 : 256;
  const bool element = rows_per_gate == 1;
  const int64_t span = element ? rows : rows_per_gate;  // rows of one gate row
  const int64_t gates = rows / span;
  BackwardPlan plan;
  // At least eight rows to a group of threads once every CU has a workgroup: each workgroup costs a
  // row of partial sums.
  const int64_t turns = ceil_div(rows, backward_rows_at_once(width));
  const int64_t wanted = std::min(most, std::max(ceil_div(turns, 8), std::min<int64_t>(turns, 256)));
  plan.splits = gates >= wanted ? 1 : ceil_div(wanted, gates);
  plan.unit_rows = ceil_div(span, plan.splits);
  plan.splits = ceil_div(span, plan.unit_rows);
  plan.units = gates * plan.splits;
  plan.groups = std::min(wanted, plan.units);
  return plan;
}

template <bool kForward>
int launch(const NormArgs& args, int dtype, int64_t groups, hipStream_t stream) {
  const int size = dtype == FHOAD_FLOAT32 ? 4 : 2;
  uintptr_t all = static_cast<uintptr_t>(args.width * size);
  for (const void* p : {args.residual, args.block, args.gate, args.weight, args.bias, args.post_weight,
                        args.post_bias, args.grad_hidden, args.grad_normed,
                        const_cast<const void*>(args.hidden), const_cast<const void*>(args.normed),
                        const_cast<const void*>(args.grad_residual), const_cast<const void*>(args.grad_block),
                        const_cast<const void*>(args.grad_gate)}) {
    all |= reinterpret_cast<uintptr_t>(p);
  }
  const bool vectors = all % 16 == 0;
  const auto go = [&](auto type, auto whole) {
    typedef decltype(type) T;
    constexpr bool kWhole = decltype(whole)::value;
    with_layout<kForward>(args.width, [&](auto threads, auto per) {
      constexpr int kThreads = decltype(threads)::value, kPer = decltype(per)::value;
      const auto run = [&](auto kernel) {
        kernel<<<static_cast<unsigned>(groups), kGroup<kThreads>, 0, stream>>>(args);
      };
      if constexpr (kForward) {
        run(norm_forward_kernel<T, kPer, kThreads, kWhole>);
      } else if (args.post_weight) {
        args.element_gate ? run(norm_backward_kernel<T, kPer, kThreads, kWhole, true, true>)
                          : run(norm_backward_kernel<T, kPer, kThreads, kWhole, true, false>);
      } else {
        args.element_gate ? run(norm_backward_kernel<T, kPer, kThreads, kWhole, false, true>)
                          : run(norm_backward_kernel<T, kPer, kThreads, kWhole, false, false>);
      }
    });
  };
  if (dtype == FHOAD_FLOAT32) {
    vectors ? go(float{}, std::true_type()) : go(float{}, std::false_type());
  } else {
    vectors ? go(__bf16{}, std::true_type()) : go(__bf16{}, std::false_type());
  }
  return check_launch(kForward ? "residual norm forward" : "residual norm backward");
}

int check_arguments(int64_t rows, int64_t width, int64_t rows_per_gate, const void* gate, int kind,
                    int dtype, const void* block, const void* post_weight, const void* post_bias) {
  if (int status = check_dtype(dtype)) return status;
  if (kind != FHOAD_RMS_NORM && kind != FHOAD_LAYER_NORM) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "kind must be FHOAD_RMS_NORM or FHOAD_LAYER_NORM");
  }
  if (rows < 0 || width < 1 || width > FHOAD_NORM_MAX_WIDTH) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "rows must be non-negative and width 1 to %d", FHOAD_NORM_MAX_WIDTH);
  }
  if (gate && (rows_per_gate < 1 || rows % rows_per_gate != 0)) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "rows must be a multiple of rows_per_gate");
  }
  if (!block && (gate || post_weight)) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "a gate or post_weight needs a block");
  }
  if (post_bias && !post_weight) return fail(FHOAD_ERROR_INVALID_VALUE, "post_bias needs post_weight");
  return FHOAD_SUCCESS;
}

}  // namespace
}  // namespace fhoad_net

using namespace fhoad_net;

extern "C" int fhoad_residual_norm_forward(const void* residual, const void* block, const void* gate,
                                           const void* weight, const void* bias,
                                           const void* post_weight, const void* post_bias,
                                           void* hidden, void* normed, float* statistics,
                                           int64_t rows, int64_t width, int64_t rows_per_gate,
                                           int kind, int dtype, double residual_scale, double eps,
                                           void* stream) {
  if (int status = check_arguments(rows, width, rows_per_gate, gate, kind, dtype, block, post_weight, post_bias)) {
    return status;
  }
  if (!(eps >= 0.0)) return fail(FHOAD_ERROR_INVALID_VALUE, "eps must be non-negative");
  if (rows == 0) return FHOAD_SUCCESS;
  if (!residual || !weight || !normed || (block && !hidden)) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "null device pointer");
  }
  if (statistics && !aligned16(statistics)) {
    return fail(FHOAD_ERROR_MISALIGNED, "statistics must be 16-byte aligned");
  }
  int cus = 0;
  if (int status = device_cus(&cus)) return status;
  NormArgs a{};
  a.residual = residual; a.block = block; a.gate = gate; a.weight = weight; a.bias = bias;
  a.post_weight = post_weight; a.post_bias = post_bias; a.hidden = hidden; a.normed = normed;
  a.statistics = statistics;
  a.rows = rows; a.width = width; a.rows_per_gate = gate ? rows_per_gate : rows;
  a.scale = static_cast<float>(residual_scale); a.eps = static_cast<float>(eps);
  a.layer = kind == FHOAD_LAYER_NORM;
  const int64_t most = static_cast<int64_t>(cus) * (width <= 1024 ? 16 : width <= 4096 ? 8 : 2);
  const int64_t groups = std::min(most, ceil_div(rows, forward_rows_at_once(width)));
  return launch<true>(a, dtype, groups, static_cast<hipStream_t>(stream));
}

extern "C" size_t fhoad_residual_norm_backward_workspace_size(int64_t rows, int64_t width,
                                                              int64_t rows_per_gate) {
  if (rows <= 0 || width <= 0) return 0;
  if (rows_per_gate < 1 || rows % rows_per_gate != 0) rows_per_gate = rows;
  const BackwardPlan plan = backward_plan(rows, width, rows_per_gate);
  return static_cast<size_t>(4 * plan.groups + (plan.splits > 1 ? plan.units : 0)) * width * sizeof(float);
}

extern "C" int fhoad_residual_norm_backward(
    const void* residual, const void* block, const void* gate, const void* weight,
    const void* post_weight, const void* post_bias, const float* statistics,
    const void* grad_hidden, const void* grad_normed, void* grad_residual, void* grad_block,
    void* grad_gate, void* grad_weight, void* grad_bias, void* grad_post_weight,
    void* grad_post_bias, void* workspace, size_t workspace_bytes, int64_t rows, int64_t width,
    int64_t rows_per_gate, int kind, int dtype, double residual_scale, void* stream) {
  if (int status = check_arguments(rows, width, rows_per_gate, gate, kind, dtype, block, post_weight, post_bias)) {
    return status;
  }
  if ((grad_gate && !gate) || (grad_block && !block) || ((grad_post_weight || grad_post_bias) && !post_weight)) {
    return fail(FHOAD_ERROR_INVALID_VALUE, "a gradient is asked for of an input that is not there");
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows == 0) {
    for (void* sum : {grad_weight, grad_bias, grad_post_weight, grad_post_bias}) {
      if (int status = zero(sum, width, dtype, s)) return status;
    }
    return FHOAD_SUCCESS;
  }
  if (!residual || !weight || !statistics) return fail(FHOAD_ERROR_INVALID_VALUE, "null device pointer");
  if (!aligned16(statistics)) return fail(FHOAD_ERROR_MISALIGNED, "statistics must be 16-byte aligned");
  if (!gate) rows_per_gate = rows;
  if (int status = check_workspace(workspace, workspace_bytes,
                                   fhoad_residual_norm_backward_workspace_size(rows, width, rows_per_gate))) {
    return status;
  }
  const BackwardPlan plan = backward_plan(rows, width, rows_per_gate);
  NormArgs a{};
  a.residual = residual; a.block = block; a.gate = gate; a.weight = weight;
  a.post_weight = post_weight; a.post_bias = post_bias;
  a.grad_hidden = grad_hidden; a.grad_normed = grad_normed; a.grad_residual = grad_residual;
  a.grad_block = grad_block; a.grad_gate = grad_gate;
  a.statistics = const_cast<float*>(statistics);
  a.partials = static_cast<float*>(workspace);
  a.rows = rows; a.width = width; a.rows_per_gate = rows_per_gate;
  a.units = plan.units; a.splits = plan.splits; a.unit_rows = plan.unit_rows;
  a.scale = static_cast<float>(residual_scale);
  a.layer = kind == FHOAD_LAYER_NORM;
  a.element_gate = gate && rows_per_gate == 1;
  a.want_sums = grad_weight || grad_bias || grad_post_weight || grad_post_bias;
  if (int status = launch<false>(a, dtype, plan.groups, s)) return status;
  const float* const partials = a.partials;
  const int64_t stride = 4 * width;
  const bool gate_sums = grad_gate && !a.element_gate && plan.splits > 1;
  const ColumnSum jobs[] = {
      {partials, grad_weight, plan.groups, stride, 0, 1},
      {partials + width, grad_bias, plan.groups, stride, 0, 1},
      {partials + 2 * width, grad_post_weight, plan.groups, stride, 0, 1},
      {partials + 3 * width, grad_post_bias, plan.groups, stride, 0, 1},
      {partials + 4 * plan.groups * width, gate_sums ? grad_gate : nullptr, plan.splits, width,
       plan.splits * width, plan.units / plan.splits},
  };
  return launch_column_sums(jobs, 5, width, dtype, s);
}
