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

constexpr int kLossThreads = 256;
constexpr int kLossWaves = kLossThreads / kWave;
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

// Maximum over a workgroup, the same in every thread.
__device__ __forceinline__ float group_max(float v, float* lds) {
  v = wave_max_f(v);
  __syncthreads();
  if (lane_id() == 0) lds[wave_id()] = v;
  __syncthreads();
  float m = lds[0];
#pragma unroll
  for (int i = 1; i < kLossWaves; ++i) m = fmaxf(m, lds[i]);
  return m;
}

template <typename T>
__global__ __launch_bounds__(kLossThreads) void loss_forward_any_kernel(LossArgs a) {
  __shared__ float lds[kLossWaves];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t t = a.target[row];
    if (t == a.ignore) {
      if (threadIdx.x == 0) a.loss[row] = 0.f;
      continue;
    }
    const T* z = static_cast<const T*>(a.z) + row * a.classes;
    float m = -INFINITY;
    for (int64_t i = threadIdx.x; i < a.classes; i += kLossThreads) m = fmaxf(m, (float)z[i]);
    m = group_max(m, lds);
    // a NaN logit, +inf, or a row of -inf alone makes the sum NaN
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < a.classes; i += kLossThreads) s += expf((float)z[i] - m);
    s = group_sum<kLossWaves>(s, lds);
    if (threadIdx.x == 0) {
      const float l = logf(s);
      const bool inside = t >= 0 && t < a.classes;
      a.loss[row] = inside ? l + (m - (float)z[t]) : NAN;
      if (a.stats) {
        a.stats[2 * row] = m;
        a.stats[2 * row + 1] = inside ? l : NAN;
      }
    }
  }
}

// The sum or mean of the rows' losses, and how many rows count (one workgroup;
// sums in 64 bits, each thread its rows in order).
constexpr int kReduceThreads = 1024;
__global__ __launch_bounds__(kReduceThreads) void loss_reduce_kernel(LossArgs a) {
  __shared__ double sums[kReduceThreads];
  __shared__ double counts[kReduceThreads];
  double s = 0.0, n = 0.0;
  for (int64_t row = threadIdx.x; row < a.rows; row += kReduceThreads) {
    s += a.loss[row];
    n += a.target[row] != a.ignore ? 1.0 : 0.0;
  }
  sums[threadIdx.x] = s;
  counts[threadIdx.x] = n;
  for (int step = kReduceThreads / 2; step > 0; step /= 2) {
    __syncthreads();
    if (threadIdx.x < step) {
      sums[threadIdx.x] += sums[threadIdx.x + step];
      counts[threadIdx.x] += counts[threadIdx.x + step];
    }
  }
  if (threadIdx.x == 0) {
    // no counted row: 0 / 0 = NaN for the mean, as its definition has it
    *a.reduced = (float)(a.reduction == kMean ? sums[0] / counts[0] : sums[0]);
    *a.count = (float)counts[0];
  }
}

template <typename T>
__global__ __launch_bounds__(kLossThreads) void loss_backward_any_kernel(LossArgs a) {
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t t = a.target[row];
    const T* z = static_cast<const T*>(a.z) + row * a.classes;
    T* dz = static_cast<T*>(a.dz) + row * a.classes;
    if (t == a.ignore) {
      for (int64_t i = threadIdx.x; i < a.classes; i += kLossThreads) dz[i] = (T)0.0f;
      continue;
    }
    const float m = a.stats[2 * row], l = a.stats[2 * row + 1];
    float c = a.grad[a.reduction == kNone ? row : 0];
    if (a.reduction == kMean) c /= *a.count;
    for (int64_t i = threadIdx.x; i < a.classes; i += kLossThreads) {
      const float p = expf(((float)z[i] - m) - l);
      dz[i] = (T)((p - (i == t ? 1.0f : 0.0f)) * c);
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

unsigned loss_groups(int64_t rows) { return (unsigned)std::min<int64_t>(rows, 1 << 20); }

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
  JN_REQUIRE(logits && target && loss && ((reduced && count) || reduction == kNone), kInvalidArgument, "null tensor pointer");
  const auto s = static_cast<hipStream_t>(stream);
  const int rc = with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    JN_PROFILE("loss_forward_any_kernel", s);
    hipLaunchKernelGGL(loss_forward_any_kernel<T>, dim3(loss_groups(rows)), dim3(kLossThreads), 0, s, a);
    JN_LAUNCH_CHECK();
    return kOk;
  });
  if (rc || reduction == kNone) return rc;
  JN_PROFILE("loss_reduce_kernel", s);
  hipLaunchKernelGGL(loss_reduce_kernel, dim3(1), dim3(kReduceThreads), 0, s, a);
  JN_LAUNCH_CHECK();
  return kOk;
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
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    JN_PROFILE("loss_backward_any_kernel", s);
    hipLaunchKernelGGL(loss_backward_any_kernel<T>, dim3(loss_groups(rows)), dim3(kLossThreads), 0, s, a);
    JN_LAUNCH_CHECK();
    return kOk;
  });
}

}  // extern "C"
