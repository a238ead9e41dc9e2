// Layer norm of rows, forward and backward, with the path scale and the state
// that a layer update carries beside it (jn_layer_norm_*).
//
//   v = scale * x,  m = mean(v),  r = 1 / sqrt(mean((v - m)^2) + eps),
//   h = (v - m) r,  y = h w + b;   state_out = tanh(scale * state)
//
//   g_w = g w;  dx = scale r (g_w - mean(g_w) - h mean(g_w h))
//   dw = sum over rows of g h,  db = sum over rows of g
//   dstate = scale (1 - tanh^2) g_state
#include "../../include/jakal_net_hip.h"
#include "jn_internal.hpp"
#include "jn_rows.hpp"

namespace jakal {
namespace {

struct NormArgs {
  const void* x;
  const void* w;    // or null (1)
  const void* b;    // or null (0)
  const void* state;  // [rows] or null
  int64_t rows, dim;
  float scale, eps;
  int state_type, param_type;
  // forward
  void* y;
  void* state_out;
  float* stats;     // [rows][2]: m, r; or null
  // backward
  const void* g;
  const void* g_state;
  void* dx;         // or null
  void* dstate;     // or null
  float* partial;   // [slabs][2][dim]
  void* dw;         // or null
  void* db;         // or null
};

// tanh and its slope 1 - tanh^2 = 4 e / (1 + e)^2 with e = exp(-2 |v|), which
// keeps its digits where tanh rounds to 1.
__device__ __forceinline__ float tanh_slope(float v) {
  const float e = expf(-2.0f * fabsf(v));
  const float d = 1.0f + e;
  return 4.0f * e / (d * d);
}

__device__ __forceinline__ void state_forward(const NormArgs& a, int64_t row) {
  store_any(a.state_out, row, a.state_type, tanhf(a.scale * load_any(a.state, row, a.state_type)));
}
__device__ __forceinline__ void state_backward(const NormArgs& a, int64_t row) {
  const float slope = tanh_slope(a.scale * load_any(a.state, row, a.state_type));
  store_any(a.dstate, row, a.state_type, a.scale * slope * load_any(a.g_state, row, a.state_type));
}

__device__ __forceinline__ float param(const void* p, int64_t i, int code, float none) {
  return p ? load_any(p, i, code) : none;
}

// Rows of any width and alignment: a workgroup a row, three passes over it.
constexpr int kAnyThreads = 256;
constexpr int kAnyWaves = kAnyThreads / kWave;

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void norm_forward_any_kernel(NormArgs a) {
  __shared__ float lds[kAnyWaves];
  const float n = (float)a.dim;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.dim;
    T* y = static_cast<T*>(a.y) + row * a.dim;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += kAnyThreads) s += a.scale * (float)x[i];
    const float m = group_sum<kAnyWaves>(s, lds) / n;
    s = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += kAnyThreads) {
      const float c = a.scale * (float)x[i] - m;
      s += c * c;
    }
    const float r = 1.0f / sqrtf(group_sum<kAnyWaves>(s, lds) / n + a.eps);
    for (int64_t i = threadIdx.x; i < a.dim; i += kAnyThreads) {
      const float h = (a.scale * (float)x[i] - m) * r;
      y[i] = (T)(h * param(a.w, i, a.param_type, 1.0f) + param(a.b, i, a.param_type, 0.0f));
    }
    if (threadIdx.x == 0) {
      if (a.stats) {
        a.stats[2 * row] = m;
        a.stats[2 * row + 1] = r;
      }
      if (a.state) state_forward(a, row);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void norm_backward_any_kernel(NormArgs a) {
  __shared__ float lds[kAnyWaves];
  const float n = (float)a.dim;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (a.dstate && threadIdx.x == 0) state_backward(a, row);
    if (!a.dx) continue;
    const T* x = static_cast<const T*>(a.x) + row * a.dim;
    const T* g = static_cast<const T*>(a.g) + row * a.dim;
    T* dx = static_cast<T*>(a.dx) + row * a.dim;
    const float m = a.stats[2 * row], r = a.stats[2 * row + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += kAnyThreads) {
      const float gw = (float)g[i] * param(a.w, i, a.param_type, 1.0f);
      s1 += gw;
      s2 += gw * ((a.scale * (float)x[i] - m) * r);
    }
    s1 = group_sum<kAnyWaves>(s1, lds) / n;
    s2 = group_sum<kAnyWaves>(s2, lds) / n;
    const float sr = a.scale * r;
    for (int64_t i = threadIdx.x; i < a.dim; i += kAnyThreads) {
      const float gw = (float)g[i] * param(a.w, i, a.param_type, 1.0f);
      const float h = (a.scale * (float)x[i] - m) * r;
      dx[i] = (T)(sr * (gw - s1 - h * s2));
    }
  }
}

// Partial column sums of g h and g: a workgroup takes 64 columns of a slab of
// rows, its four waves every fourth row.
template <typename T>
__global__ __launch_bounds__(kAnyThreads) void norm_columns_any_kernel(NormArgs a, int64_t slab_rows) {
  __shared__ float lds[2][kAnyWaves][kWave];
  const int64_t c = (int64_t)blockIdx.x * kWave + lane_id();
  const int64_t r0 = (int64_t)blockIdx.y * slab_rows;
  const int64_t r1 = r0 + slab_rows < a.rows ? r0 + slab_rows : a.rows;
  float sw = 0.f, sb = 0.f;
  if (c < a.dim) {
    for (int64_t row = r0 + wave_id(); row < r1; row += kAnyWaves) {
      const float g = (float)static_cast<const T*>(a.g)[row * a.dim + c];
      const float x = (float)static_cast<const T*>(a.x)[row * a.dim + c];
      sw += g * ((a.scale * x - a.stats[2 * row]) * a.stats[2 * row + 1]);
      sb += g;
    }
  }
  lds[0][wave_id()][lane_id()] = sw;
  lds[1][wave_id()][lane_id()] = sb;
  __syncthreads();
  if (wave_id() < 2 && c < a.dim) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kAnyWaves; ++i) s += lds[wave_id()][i][lane_id()];
    a.partial[((int64_t)blockIdx.y * 2 + wave_id()) * a.dim + c] = s;
  }
}

// The slabs' partial sums, in slab order.
__global__ __launch_bounds__(kAnyThreads) void norm_columns_finish_kernel(NormArgs a, int slabs) {
  const int64_t c = (int64_t)blockIdx.x * kAnyThreads + threadIdx.x;
  if (c >= a.dim) return;
  float sw = 0.f, sb = 0.f;
  for (int s = 0; s < slabs; ++s) {
    sw += a.partial[(int64_t)s * 2 * a.dim + c];
    sb += a.partial[((int64_t)s * 2 + 1) * a.dim + c];
  }
  if (a.dw) store_any(a.dw, c, a.param_type, sw);
  if (a.db) store_any(a.db, c, a.param_type, sb);
}

// Row slabs of the column sums.
constexpr int64_t kSlabs = 64;
int64_t slab_count(int64_t rows) { return std::min<int64_t>(kSlabs, (rows + 15) / 16); }

int64_t row_groups(int64_t rows) { return std::min<int64_t>(rows, 1 << 20); }

int check_norm(const NormArgs& a, int32_t type, int32_t state_type, int32_t param_type) {
  JN_REQUIRE(known_type(type) && known_type(state_type) && known_type(param_type), kInvalidArgument,
             "layer norm: element types are 0 (fp32), 1 (bf16) and 2 (fp16), got %d, %d, %d", (int)type,
             (int)state_type, (int)param_type);
  JN_REQUIRE(param_type == kTypeF32 || param_type == type, kInvalidArgument,
             "layer norm: parameters are fp32 or of the rows' type (types %d and %d)", (int)param_type, (int)type);
  JN_REQUIRE(a.rows >= 0 && a.dim >= 1 && a.dim < (1LL << 28) && a.rows <= (1LL << 40) / a.dim, kInvalidArgument,
             "layer norm needs rows >= 0, 1 <= dim < 2^28 and at most 2^40 elements (rows=%lld, dim=%lld)",
             (long long)a.rows, (long long)a.dim);
  return kOk;
}

}  // namespace
}  // namespace jakal

using namespace jakal;

extern "C" {

int jn_layer_norm_forward(const void* state, const void* x, const void* weight, const void* bias, int64_t rows,
                          int64_t dim, float scale, float eps, int32_t type, int32_t state_type, int32_t param_type,
                          void* state_out, void* y, float* stats, jn_stream_t stream) {
  NormArgs a{};
  a.x = x, a.w = weight, a.b = bias, a.state = state, a.rows = rows, a.dim = dim, a.scale = scale, a.eps = eps;
  a.state_type = state_type, a.param_type = param_type, a.y = y, a.state_out = state_out, a.stats = stats;
  if (const int rc = check_norm(a, type, state_type, param_type)) return rc;
  JN_REQUIRE(eps >= 0.0f, kInvalidArgument, "layer norm: eps must not be negative");
  if (rows == 0) return kOk;
  JN_REQUIRE(x && y && (!state || state_out), kInvalidArgument, "null tensor pointer");
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    JN_PROFILE("norm_forward_any_kernel", s);
    hipLaunchKernelGGL(norm_forward_any_kernel<T>, dim3((unsigned)row_groups(rows)), dim3(kAnyThreads), 0, s, a);
    JN_LAUNCH_CHECK();
    return kOk;
  });
}

size_t jn_layer_norm_backward_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows < 1 || dim < 1 || dim >= (1LL << 28)) return 0;
  return (size_t)slab_count(rows) * 2 * dim * sizeof(float);
}

int jn_layer_norm_backward(const void* state, const void* x, const void* weight, const float* stats,
                           const void* grad_state_out, const void* grad_y, int64_t rows, int64_t dim, float scale,
                           int32_t type, int32_t state_type, int32_t param_type, void* grad_state, void* grad_x,
                           void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                           jn_stream_t stream) {
  NormArgs a{};
  a.x = x, a.w = weight, a.state = state, a.rows = rows, a.dim = dim, a.scale = scale;
  a.state_type = state_type, a.param_type = param_type, a.stats = const_cast<float*>(stats);
  a.g = grad_y, a.g_state = grad_state_out, a.dx = grad_x, a.dstate = grad_state;
  a.partial = static_cast<float*>(workspace), a.dw = grad_weight, a.db = grad_bias;
  if (const int rc = check_norm(a, type, state_type, param_type)) return rc;
  JN_REQUIRE(rows >= 1, kInvalidArgument, "layer norm backward needs at least one row");
  const bool columns = grad_weight || grad_bias;
  JN_REQUIRE(!grad_state || (state && grad_state_out), kInvalidArgument, "null tensor pointer");
  JN_REQUIRE((!grad_x && !columns) || (x && stats && grad_y), kInvalidArgument, "null tensor pointer");
  const size_t need = columns ? jn_layer_norm_backward_workspace_bytes(rows, dim) : 0;
  JN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), kWorkspaceTooSmall,
             "layer norm backward needs %zu workspace bytes, got %zu", need, workspace_bytes);
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (grad_x || grad_state) {
      JN_PROFILE("norm_backward_any_kernel", s);
      hipLaunchKernelGGL(norm_backward_any_kernel<T>, dim3((unsigned)row_groups(rows)), dim3(kAnyThreads), 0, s, a);
      JN_LAUNCH_CHECK();
    }
    if (columns) {
      const int64_t slabs = slab_count(rows);
      const int64_t slab_rows = (rows + slabs - 1) / slabs;
      {
        JN_PROFILE("norm_columns_any_kernel", s);
        hipLaunchKernelGGL(norm_columns_any_kernel<T>, dim3((unsigned)((dim + kWave - 1) / kWave), (unsigned)slabs),
                           dim3(kAnyThreads), 0, s, a, slab_rows);
        JN_LAUNCH_CHECK();
      }
      JN_PROFILE("norm_columns_finish_kernel", s);
      hipLaunchKernelGGL(norm_columns_finish_kernel, dim3((unsigned)((dim + kAnyThreads - 1) / kAnyThreads)),
                         dim3(kAnyThreads), 0, s, a, (int)slabs);
      JN_LAUNCH_CHECK();
    }
    return kOk;
  });
}

}  // extern "C"
