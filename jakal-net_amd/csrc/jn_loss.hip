// Cross entropy of logit rows against class indices, and its gradient
// (jn_cross_entropy_*).
//
//   M = max_j z_j,  L = log sum_j exp(z_j - M),  loss = L + (M - z_t)
//   dz_j = (exp((z_j - M) - L) - [j = t]) c,
//   c = grad / count (mean), grad (sum), grad of the row (none)
//
// M and L are kept apart for the backward: z - M is exact or nearly so, while
// M + L would lose the digits of L under a large M.  Rows whose target is
// ignore_index read no logits: loss 0, gradient 0.  A target outside the
// classes reads nothing out of range and makes its row's loss and gradient NaN.
#include "../../include/jakal_net_hip.h"
#include "jn_internal.hpp"
#include "jn_rows.hpp"

namespace jakal {
namespace {

constexpr int kNone = 0, kMean = 2;  // reductions (1: sum)

struct LossArgs {
  const void* z;
  const int64_t* target;
  int64_t rows, classes, ignore;
  float* loss;       // [rows]
  float* stats;      // [rows][2]: M, L
  int reduction;
  float* reduced;    // the reduced loss
  float* count;      // the rows that count
  const float* grad;  // one, or [rows] with reduction none
  void* dz;
};

// A row's elements as its memory has them: whole aligned packs of W elements,
// and up to W - 1 single ones on either side, so that rows may start anywhere
// (an odd vocabulary) and still move 16 bytes a lane.
template <typename T>
struct RowSpan {
  static constexpr int W = 16 / sizeof(T);
  int head, tail;  // single elements before and after the packs
  int packs;
  int64_t n;

  __device__ RowSpan(const T* row, int64_t classes) : n(classes) {
    const int off = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    head = classes < off ? (int)classes : off;
    packs = (int)((classes - head) / W);
    tail = (int)(classes - head - (int64_t)packs * W);
  }
  // the single element that thread t takes, or -1: the head's by the first threads, the tail's by those from 32
  __device__ int64_t single(int t) const {
    if (t < head) return t;
    return t >= 32 && t - 32 < tail ? n - tail + t - 32 : -1;
  }
  __device__ int64_t element(int pack) const { return head + (int64_t)pack * W; }
};

// A running maximum m and the sum s of exponentials below it.  s is 0 under a
// maximum of -inf, and NaN once a NaN or +inf was met.
//
// The sums take the hardware's 2^t of t = x log2(e), whose rounding makes |x| / 2
// ulps of a term.  Of log s that is 2^-24 times the mean of |x| under the softmax
// at most, and that mean is log(classes) at most: an ulp of the loss where all
// terms round the same way, less where they differ.  8,192 rows of 16,384 bf16
// classes, a fifth ignored, take 41 us so, 68 with expf() and 52 with exp_of().
struct LogSum {
  float m = -INFINITY, s = 0.f;

  __device__ __forceinline__ void join(float m2, float s2) {
    const float top = fmaxf(m, m2);
    s = (m == top ? s : s * __expf(m - top)) + (m2 == top ? s2 : s2 * __expf(m2 - top));
    m = top;
  }
  __device__ __forceinline__ void add(float z) { join(fmaxf(z, -INFINITY), z == -INFINITY ? 0.f : __expf(z - z)); }
};

// One row by THREADS threads: each reads its packs kPacks at a time, takes their
// maximum and then their exponentials from registers (one rescaling of its sum
// for 16 kPacks bytes); the threads' pairs join at the end, in every thread.
constexpr int kPacks = 8;
template <typename T, int THREADS>
__device__ __forceinline__ LogSum row_log_sum(const T* z, int64_t classes, float (*lds)[2]) {
  constexpr int W = RowSpan<T>::W, kWaves = THREADS / kWave;
  const int t = THREADS == kWave ? lane_id() : (int)threadIdx.x;
  const RowSpan<T> span(z, classes);
  LogSum sum;
  const int64_t one = span.single(t);
  if (one >= 0) sum.add((float)z[one]);
  for (int first = t; first < span.packs; first += THREADS * kPacks) {
    Raw<T, W> raw[kPacks];
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      if (first + i * THREADS < span.packs) raw[i].load(z + span.element(first + i * THREADS));
    }
    float m = sum.m;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      if (first + i * THREADS >= span.packs) continue;
      float v[W];
      raw[i].unpack(v);
#pragma unroll
      for (int j = 0; j < W; ++j) m = fmaxf(m, v[j]);
    }
    const float base = m == -INFINITY ? 0.f : m;  // exp(-inf - 0) = 0
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      if (first + i * THREADS >= span.packs) continue;
      float v[W];
      raw[i].unpack(v);
#pragma unroll
      for (int j = 0; j < W; ++j) s += __expf(v[j] - base);
    }
    sum.join(m, s);
  }
  const float top = wave_max_f(sum.m);
  sum.s = wave_sum(sum.m == top ? sum.s : sum.s * __expf(sum.m - top));
  sum.m = top;
  if constexpr (kWaves > 1) {
    __syncthreads();  // an earlier row's readers are done
    if (lane_id() == 0) {
      lds[wave_id()][0] = sum.m;
      lds[wave_id()][1] = sum.s;
    }
    __syncthreads();
    sum = LogSum{};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum.join(lds[i][0], lds[i][1]);
  }
  return sum;
}

// THREADS = 64: a wave a row, four rows a workgroup; else a workgroup a row.
// Bound by the read of the logits: 6,550 rows of 16,384 bf16 (215 MB) in 40 us,
// 5.4 TB/s; with the exponentials left out it takes as long.  Rows wait to be
// taken by a free workgroup: held by persistent ones, with the next row's loads
// in flight, they took 67 us, since ignored rows leave some idle.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS == kWave ? 4 * kWave : THREADS) void loss_forward_kernel(LossArgs a) {
  constexpr int kRows = THREADS == kWave ? 4 : 1;
  __shared__ float lds[THREADS / kWave][2];
  const int64_t step = (int64_t)gridDim.x * kRows;
  for (int64_t row = (int64_t)blockIdx.x * kRows + (kRows > 1 ? wave_id() : 0); row < a.rows; row += step) {
    const int64_t t = a.target[row];
    const bool writes = (THREADS == kWave ? lane_id() : (int)threadIdx.x) == 0;
    if (t == a.ignore) {
      if (writes) a.loss[row] = 0.f;
      continue;
    }
    const T* z = static_cast<const T*>(a.z) + row * a.classes;
    const bool inside = t >= 0 && t < a.classes;
    const float zt = inside ? (float)z[t] : NAN;
    const LogSum sum = row_log_sum<T, THREADS>(z, a.classes, lds);
    if (writes) {
      const float l = logf(sum.s);
      a.loss[row] = l + (sum.m - zt);
      if (a.stats) {
        a.stats[2 * row] = sum.m;
        a.stats[2 * row + 1] = inside ? l : NAN;
      }
    }
  }
}

__device__ __forceinline__ void write_reduced(const LossArgs& a, double s, double n) {
  // no counted row: 0 / 0 = NaN for the mean, as its definition has it
  *a.reduced = (float)(a.reduction == kMean ? s / n : s);
  *a.count = (float)n;
}

// Few logits in one launch: a workgroup of sixteen waves takes all rows, a wave
// each, and reduces their losses.
constexpr int kSmallWaves = 16;
template <typename T>
__global__ __launch_bounds__(kSmallWaves* kWave) void loss_small_kernel(LossArgs a) {
  __shared__ double lds[kSmallWaves][2];
  double s = 0.0, n = 0.0;
  if (const int row = wave_id(); row < a.rows) {
    const int64_t t = a.target[row];
    const bool counts = t != a.ignore, inside = t >= 0 && t < a.classes;
    float loss = 0.f;
    if (counts) {
      const T* z = static_cast<const T*>(a.z) + (int64_t)row * a.classes;
      const float zt = inside ? (float)z[t] : NAN;
      const LogSum sum = row_log_sum<T, kWave>(z, a.classes, nullptr);
      const float l = logf(sum.s);
      loss = l + (sum.m - zt);
      if (a.stats && lane_id() == 0) {
        a.stats[2 * row] = sum.m;
        a.stats[2 * row + 1] = inside ? l : NAN;
      }
    }
    if (lane_id() == 0) a.loss[row] = loss;
    s = loss;
    n = counts ? 1.0 : 0.0;
  }
  if (lane_id() == 0) {
    lds[wave_id()][0] = s;
    lds[wave_id()][1] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = n = 0.0;
    for (int i = 0; i < kSmallWaves; ++i) {
      s += lds[i][0];
      n += lds[i][1];
    }
    write_reduced(a, s, n);
  }
}

// The sum or mean of the rows' losses, and how many rows count (sums in 64 bits,
// each thread its rows in order).  One workgroup up to kOneGroupRows rows, else
// many that leave a pair of sums each in `parts` for a launch of one to join: 8,192
// rows 4.2 us, 32,768 7.8 against 8.0, 65,536 12.9 against 8.1, 2^20 169 against 9.2.
constexpr int kReduceThreads = 1024, kReduceWaves = kReduceThreads / kWave;
constexpr int64_t kOneGroupRows = 32768;
constexpr int64_t kGroupRows = 4096;  // rows of a workgroup, at least
constexpr int64_t kMaxReduceGroups = 256;

__device__ __forceinline__ void join_sums(double& s, double& n, double (*lds)[2]) {
  for (int step = 1; step < kWave; step *= 2) {
    s += __shfl_xor(s, step);
    n += __shfl_xor(n, step);
  }
  if (lane_id() == 0) {
    lds[wave_id()][0] = s;
    lds[wave_id()][1] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = n = 0.0;
    for (int i = 0; i < kReduceWaves; ++i) {
      s += lds[i][0];
      n += lds[i][1];
    }
  }
}

__global__ __launch_bounds__(kReduceThreads) void loss_reduce_kernel(LossArgs a, double* parts) {
  __shared__ double lds[kReduceWaves][2];
  double s = 0.0, n = 0.0;
  const int64_t step = (int64_t)gridDim.x * kReduceThreads;
#pragma unroll 4
  for (int64_t row = (int64_t)blockIdx.x * kReduceThreads + threadIdx.x; row < a.rows; row += step) {
    s += a.loss[row];
    n += a.target[row] != a.ignore ? 1.0 : 0.0;
  }
  join_sums(s, n, lds);
  if (threadIdx.x != 0) return;
  if (parts) {
    parts[2 * blockIdx.x] = s;
    parts[2 * blockIdx.x + 1] = n;
  } else {
    write_reduced(a, s, n);
  }
}

__global__ __launch_bounds__(kReduceThreads) void loss_join_kernel(LossArgs a, const double* parts, int count) {
  __shared__ double lds[kReduceWaves][2];
  const bool has = (int)threadIdx.x < count;  // (count <= kMaxReduceGroups)
  double s = has ? parts[2 * threadIdx.x] : 0.0, n = has ? parts[2 * threadIdx.x + 1] : 0.0;
  join_sums(s, n, lds);
  if (threadIdx.x == 0) write_reduced(a, s, n);
}

int64_t reduce_groups(int64_t rows) {
  return rows <= kOneGroupRows ? 1 : std::min((rows + kGroupRows - 1) / kGroupRows, kMaxReduceGroups);
}

int launch_reduce(const LossArgs& a, double* parts, hipStream_t s) {
  const int64_t groups = parts ? reduce_groups(a.rows) : 1;
  {
    JN_PROFILE("loss_reduce_kernel", s);
    hipLaunchKernelGGL(loss_reduce_kernel, dim3((unsigned)groups), dim3(kReduceThreads), 0, s, a,
                       groups > 1 ? parts : nullptr);
    JN_LAUNCH_CHECK();
  }
  if (groups == 1) return kOk;
  JN_PROFILE("loss_join_kernel", s);
  hipLaunchKernelGGL(loss_join_kernel, dim3(1), dim3(kReduceThreads), 0, s, a, parts, (int)groups);
  JN_LAUNCH_CHECK();
  return kOk;
}

// e^x for x <= 0 (or NaN), to 1.2 ulps: the hardware's 2^t of t = x log2(e),
// times e^(what the rounding of t lost), which is 1 + that; without it x = -80
// is off by 40 ulps.  Below -150 the result is 0, and -inf has no rounding to
// give back.  The fp32 gradient takes this (8,192 x 2,048 in 19.1 us either way,
// 1,531 x 4,099 in 9.1 against 8.7; expf() 19.5 and 9.1).  Half-precision ones
// round to 2^-8 or 2^-11 of their value behind it, a hundred times what __expf
// loses at -80, and would pay 11.4 us instead of 9.5 at 1,024 x 16,384 bf16.
__device__ __forceinline__ float exp_of(float x) {
  constexpr float kLog2E = 0x1.715476p+0f, kLog2ELow = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;  // log2(e) = the two's sum
  x = x < -150.0f ? -150.0f : x;
  const float t = x * kLog2E;
  const float lost = fmaf(x, kLog2ELow, fmaf(x, kLog2E, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  return fmaf(p, lost * kLn2, p);
}

// The gradient of a stretch of a row: kPacks packs a thread (and the row's
// single elements, with its first stretch).  W = 1 where the gradient's rows do
// not start on 16 bytes where the logits' do.  The logits are read for the last
// time and the gradient is as large as they are: both go past the caches.  The
// forward, the backward and a product that reads the gradient, bf16 logits of
// 16,384 classes, so and with ordinary accesses: 1,024 rows 73 and 75 us, 4,096
// 149 and 173, 8,192 339 and 386.  By itself 8,192 rows, a fifth ignored, take
// 67 us (485 MB, 7.3 TB/s).
template <typename T, int W>
__device__ __forceinline__ void loss_gradient(T* dz, int64_t e, int64_t t, float m, float l, float c,
                                              const Raw<T, W>& raw) {
  float v[W];
  raw.unpack(v);
#pragma unroll
  for (int j = 0; j < W; ++j) {
    const float x = (v[j] - m) - l;
    v[j] = std::is_same_v<T, float> ? exp_of(x) : __expf(x);
  }
  const int64_t hot = t - e;
  if (hot >= 0 && hot < W) {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] -= j == hot ? 1.0f : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] *= c;
  store_raw<T, W, true>(dz + e, v);
}

template <typename T, int THREADS, bool PACKED>
__global__ __launch_bounds__(THREADS == kWave ? 4 * kWave : THREADS) void loss_backward_kernel(LossArgs a) {
  constexpr int kRows = THREADS == kWave ? 4 : 1;
  constexpr int W = PACKED ? RowSpan<T>::W : 1;
  constexpr int64_t kStretch = (int64_t)THREADS * kPacks;
  const int thread = THREADS == kWave ? lane_id() : (int)threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * kRows;
  for (int64_t row = (int64_t)blockIdx.x * kRows + (kRows > 1 ? wave_id() : 0); row < a.rows; row += step) {
    const int64_t t = a.target[row];
    const T* z = static_cast<const T*>(a.z) + row * a.classes;
    T* dz = static_cast<T*>(a.dz) + row * a.classes;
    const bool ignored = t == a.ignore;
    const float m = ignored ? 0.f : a.stats[2 * row], l = ignored ? 0.f : a.stats[2 * row + 1];
    float c = ignored ? 0.f : a.grad[a.reduction == kNone ? row : 0];
    if (!ignored && a.reduction == kMean) c /= *a.count;
    const RowSpan<T> span(z, a.classes);
    const int64_t packs = PACKED ? span.packs : a.classes, head = PACKED ? span.head : 0;
    if (PACKED && blockIdx.y == 0) {
      const int64_t one = span.single(thread);
      if (one >= 0) {
        Raw<T, 1> raw;
        if (ignored) dz[one] = (T)0.0f;
        else raw.load(z + one), loss_gradient<T, 1>(dz, one, t, m, l, c, raw);
      }
    }
    for (int64_t first = blockIdx.y * kStretch + thread; first < packs; first += gridDim.y * kStretch) {
      Raw<T, W> raw[kPacks];
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        const int64_t p = first + i * THREADS;
        if (p < packs && !ignored) raw[i].template load<true>(z + head + p * W);
        else raw[i].clear();
      }
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        const int64_t p = first + i * THREADS;
        if (p >= packs) continue;
        if (ignored) raw[i].template store<true>(dz + head + p * W);
        else loss_gradient<T, W>(dz, head + p * W, t, m, l, c, raw[i]);
      }
    }
  }
}

int check_loss(const LossArgs& a, int32_t type) {
  JN_REQUIRE(known_type(type), kInvalidArgument, "cross entropy: the element type is 0 (fp32), 1 (bf16) or 2 (fp16), "
             "got %d", (int)type);
  JN_REQUIRE(a.rows >= 1 && a.classes >= 1 && a.classes < (1LL << 31) && a.rows <= (1LL << 40) / a.classes,
             kInvalidArgument,
             "cross entropy needs rows >= 1, 1 <= classes < 2^31 and at most 2^40 logits (rows=%lld, classes=%lld)",
             (long long)a.rows, (long long)a.classes);
  JN_REQUIRE(a.reduction >= kNone && a.reduction <= kMean, kInvalidArgument,
             "cross entropy: the reduction is 0 (none), 1 (sum) or 2 (mean), got %d", a.reduction);
  return kOk;
}

// Rows of up to kWaveClasses take a wave each; so do rows of up to `chunks` times
// a wave's kPacks packs a lane where they are many.  Longer ones take a
// workgroup, in the forward of 1024 threads where there are too few rows to fill
// the CUs otherwise.  8,192 rows, wave against workgroup, forward and backward:
// 1,100 bf16 12.6 and 11.8 us against 26.4 and 19.2, 4,096 bf16 19.9 and 28.6
// against 32.8 and 29.8, 8,192 bf16 31.0 and 56.7 against 38.3 and 48.9 (two
// chunks); fp32 2,048 17.6 and 28.0 against 20.8 and 28.1, 4,099 30.3 and 56.9
// against 28.2 and 47.5 (two chunks); at 1,024 rows they are equal.
// One launch by one workgroup where each of its waves has one row at most, short
// enough for a wave (a captured call, one launch against two, fp32 and bf16: 16 x
// 64 2.9 and 3.7 against 4.9 and 5.6 us, 16 x 4,000 5.5 and 5.3 against 6.4 and
// 6.5, 8 x 8,000 5.9 and 5.8 against 6.4 and 6.9; two rows a wave, 32 x 1,000,
// 5.1 and 6.3 against 5.1 and 5.3, 64 x 1,000 8.5 and 10.5 against 5.1 and 5.3;
// longer rows, 4 x 16,000, 8.5 and 7.1 against 6.6 and 6.9, 1 x 64,000 27 and 20
// against 8.4 and 8.1).  The second launch costs the host 4 us.
constexpr int64_t kSmallBytes = 256 << 10;
constexpr int64_t kSmallRowBytes = 32 << 10;
constexpr int64_t kWaveClasses = 1024;
constexpr int64_t kWaveRows = 1024;
constexpr int64_t kFewRows = 512;

template <typename T>
bool wave_rows(const LossArgs& a, int chunks) {
  return a.classes <= kWaveClasses ||
         (a.rows >= kWaveRows && a.classes <= (int64_t)chunks * kWave * kPacks * RowSpan<T>::W);
}

template <typename T>
int launch_loss_forward(const LossArgs& a, hipStream_t s) {
  JN_PROFILE("loss_forward_kernel", s);
  if (wave_rows<T>(a, 4 / sizeof(T))) {
    const unsigned grid = (unsigned)std::min<int64_t>((a.rows + 3) / 4, 1 << 20);
    hipLaunchKernelGGL((loss_forward_kernel<T, kWave>), dim3(grid), dim3(4 * kWave), 0, s, a);
  } else if (a.rows < kFewRows) {
    hipLaunchKernelGGL((loss_forward_kernel<T, 1024>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
  } else {
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 1 << 20);
    hipLaunchKernelGGL((loss_forward_kernel<T, 256>), dim3(grid), dim3(256), 0, s, a);
  }
  JN_LAUNCH_CHECK();
  return kOk;
}

template <typename T, bool PACKED>
int launch_loss_backward(const LossArgs& a, hipStream_t s) {
  JN_PROFILE("loss_backward_kernel", s);
  if (wave_rows<T>(a, 1)) {
    const unsigned grid = (unsigned)std::min<int64_t>((a.rows + 3) / 4, 1 << 20);
    hipLaunchKernelGGL((loss_backward_kernel<T, kWave, PACKED>), dim3(grid), dim3(4 * kWave), 0, s, a);
  } else {
    const int64_t stretch = 256 * kPacks * (PACKED ? RowSpan<T>::W : 1);
    const unsigned parts = (unsigned)std::min<int64_t>((a.classes + stretch - 1) / stretch, 1024);
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 1 << 20);
    hipLaunchKernelGGL((loss_backward_kernel<T, 256, PACKED>), dim3(grid, parts), dim3(256), 0, s, a);
  }
  JN_LAUNCH_CHECK();
  return kOk;
}

}  // namespace
}  // namespace jakal

using namespace jakal;

extern "C" {

int jn_cross_entropy_forward(const void* logits, const int64_t* target, int64_t rows, int64_t classes,
                             int64_t ignore_index, int32_t reduction, int32_t type, float* loss, float* stats,
                             float* reduced, float* count, jn_stream_t stream) {
  LossArgs a{};
  a.z = logits, a.target = target, a.rows = rows, a.classes = classes, a.ignore = ignore_index;
  a.reduction = reduction, a.loss = loss, a.stats = stats, a.reduced = reduced;
  a.count = count;
  if (const int rc = check_loss(a, type)) return rc;
  JN_REQUIRE(logits && target && loss && ((reduced && count) || reduction == kNone), kInvalidArgument,
             "null tensor pointer");
  const auto s = static_cast<hipStream_t>(stream);
  const int64_t row_bytes = classes * type_bytes(type);
  const bool small = reduction != kNone && rows <= kSmallWaves && row_bytes <= kSmallRowBytes &&
                     rows * row_bytes <= kSmallBytes;
  const int rc = with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (!small) return launch_loss_forward<T>(a, s);
    JN_PROFILE("loss_small_kernel", s);
    hipLaunchKernelGGL(loss_small_kernel<T>, dim3(1), dim3(kSmallWaves * kWave), 0, s, a);
    JN_LAUNCH_CHECK();
    return kOk;
  });
  if (rc || reduction == kNone || small) return rc;
  return launch_reduce(a, nullptr, s);
}

size_t jn_cross_entropy_reduce_workspace_bytes(int64_t rows) {
  const int64_t groups = rows < 1 ? 1 : reduce_groups(rows);
  return groups == 1 ? 0 : (size_t)groups * 2 * sizeof(double);
}

int jn_cross_entropy_reduce(const float* loss, const int64_t* target, int64_t rows, int64_t ignore_index,
                            int32_t reduction, float* reduced, float* count, void* workspace, size_t workspace_bytes,
                            jn_stream_t stream) {
  LossArgs a{};
  a.loss = const_cast<float*>(loss), a.target = target, a.rows = rows, a.classes = 1, a.ignore = ignore_index;
  a.reduction = reduction, a.reduced = reduced, a.count = count;
  if (const int rc = check_loss(a, kTypeF32)) return rc;
  JN_REQUIRE(reduction != kNone, kInvalidArgument, "cross entropy: the reduction is 1 (sum) or 2 (mean) here");
  JN_REQUIRE(loss && target && reduced && count, kInvalidArgument, "null tensor pointer");
  const size_t need = jn_cross_entropy_reduce_workspace_bytes(rows);
  JN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), kWorkspaceTooSmall,
             "the reduction of %lld losses needs %zu workspace bytes, got %zu", (long long)rows, need, workspace_bytes);
  return launch_reduce(a, need ? static_cast<double*>(workspace) : nullptr, static_cast<hipStream_t>(stream));
}

int jn_cross_entropy_backward(const void* logits, const int64_t* target, const float* stats, const float* count,
                              const float* grad_loss, int64_t rows, int64_t classes, int64_t ignore_index,
                              int32_t reduction, int32_t type, void* grad_logits, jn_stream_t stream) {
  LossArgs a{};
  a.z = logits, a.target = target, a.rows = rows, a.classes = classes, a.ignore = ignore_index;
  a.reduction = reduction, a.stats = const_cast<float*>(stats), a.count = const_cast<float*>(count);
  a.grad = grad_loss, a.dz = grad_logits;
  if (const int rc = check_loss(a, type)) return rc;
  JN_REQUIRE(logits && target && stats && grad_loss && grad_logits && (count || reduction != kMean),
             kInvalidArgument, "null tensor pointer");
  const auto s = static_cast<hipStream_t>(stream);
  const bool packed =
      ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad_logits)) & 15) == 0;
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    return packed ? launch_loss_backward<T, true>(a, s) : launch_loss_backward<T, false>(a, s);
  });
}

}  // extern "C"
