// Microscaled tensors made and read (jn_mx_quantize, jn_mx_dequantize), and the
// GELU whose input is kept in e4m3 for its backward (jn_gelu_*).
//
//   gelu(x) = x Phi(x);  gelu'(x) = Phi(x) + x phi(x), taken at the kept x
//   Phi(x) = (1 + erf(x / sqrt 2)) / 2,  phi(x) = exp(-x^2 / 2) / sqrt(2 pi)
#include "../../include/jakal_net_hip.h"
#include "jn_internal.hpp"
#include "jn_mx.hpp"

namespace jakal {
namespace {

struct UnitArgs {
  const void* x;   // read: elements, or null
  void* y;         // written: elements, or null
  uint8_t* codes;  // or null
  uint8_t* scales;
  int64_t rows, dim;
  int64_t units;      // of all rows
  int64_t row_units;  // of one
  int64_t first;      // of this launch
};

// A workgroup takes 256 units in a row; where rows are whole runs they are one long row.
struct UnitPlace {
  int64_t unit, row, e;
  __device__ explicit UnitPlace(const UnitArgs& a) {
    unit = a.first + (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (a.rows == 1) row = 0, e = unit * 8;
    else if (a.units < (int64_t(1) << 32)) {
      const uint32_t r = (uint32_t)unit / (uint32_t)a.row_units;
      row = r, e = (int64_t)((uint32_t)unit - r * (uint32_t)a.row_units) * 8;
    } else {
      row = unit / a.row_units, e = (unit - row * a.row_units) * 8;
    }
  }
};

constexpr float kRsqrt2 = 0.70710678118654752f, kRsqrt2Pi = 0.39894228040143268f;

// Phi(x), and phi(x) sqrt(2 pi) where the slope needs it.  fp32 takes the library's error
// function.  Half precision has less time for it (one element's error function and
// exponential cost as much as its bytes: 8,192 x 2,048 bf16 forward 19.0 and backward 24.8
// us), and takes the tail of the distribution, which keeps its digits on both sides:
//   Phi(-|x|) = exp(-x^2 / 2) t Q(t) / 2,  t = 1 / (1 + |x| / sqrt 8)
// the form of Hastings' approximations of the error function (Abramowitz and Stegun,
// 7.1.25 to 7.1.28).  Q is the polynomial of degree 8 for which the largest relative
// difference of t Q(t) and exp(z^2) erfc(z), z = |x| / sqrt 2 up to 10, is least (it
// is reached ten times, in turn above and below): 7.4e-8 with the coefficients rounded as below,
// 3.5e-7 as computed.  The exponential's argument adds x^2 2^-24 (8e-6 at x = -13).
template <typename T>
__device__ __forceinline__ float normal_cdf(float x, float& dense) {
  if constexpr (sizeof(T) == 4) {
    dense = expf(-0.5f * x * x);
    return 0.5f * (1.0f + erff(x * kRsqrt2));
  } else {
    dense = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
    const float t = __builtin_amdgcn_rcpf(1.0f + fabsf(x) * (0.5f * kRsqrt2));
    constexpr float q[9] = {0.282086432f, 0.282375246f, 0.243104205f, 0.202685177f, -0.0266217813f, 0.278061688f, -0.487195253f, 0.28457278f, -0.0590685233f};
    float p = q[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) p = p * t + q[i];
    const float tail = 0.5f * dense * t * p;
    return x < 0.f ? tail : 1.0f - tail;
  }
}
template <typename T>
__device__ __forceinline__ float gelu_f(float x) {
  float dense;
  return x * normal_cdf<T>(x, dense);
}
template <typename T>
__device__ __forceinline__ float gelu_slope(float x) {
  float dense;
  const float cdf = normal_cdf<T>(x, dense);
  return cdf + x * (kRsqrt2Pi * dense);
}

// The four below move bytes: a thread has a unit of eight elements, four threads a run,
// whose largest magnitude meets in the quad's lanes; no LDS, no loop.  16,384 x 2,048 bf16
// to e2m1 15 us (85 MB, 5.7 TB/s) and back 18.6 (4.6); GELU of 8,192 x 2,048 bf16 19 us
// forward (84 MB, 4.4 TB/s) and 18.5 backward (4.6), where the polynomial is as long as the
// bytes; a device copy reaches 4.8 TB/s.  64 x 512 fp32 2.4 us, one launch's latency.
template <typename T, int FORM, bool PACKED>
__global__ __launch_bounds__(256) void mx_quantize_kernel(UnitArgs a) {
  const UnitPlace at(a);
  if (at.unit >= a.units) return;  // whole quads
  float v[8];
  load_unit<T, PACKED>(static_cast<const T*>(a.x) + at.row * a.dim, at.e, a.dim, v);
  uint32_t code[2];
  const int s = mx_encode<FORM>(v, code);
  mx_store<FORM>(a.codes, a.scales, at.unit, code, s);
}

template <typename T, int FORM, bool PACKED>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(UnitArgs a) {
  const UnitPlace at(a);
  if (at.unit >= a.units) return;
  float v[8];
  mx_load<FORM>(a.codes, a.scales, at.unit, v);
  store_unit<T, PACKED>(static_cast<T*>(a.y) + at.row * a.dim, at.e, a.dim, v);
}

// y = gelu(x), and x kept where there is somewhere to keep it.
template <typename T, bool PACKED>
__global__ __launch_bounds__(256) void gelu_forward_kernel(UnitArgs a) {
  const UnitPlace at(a);
  if (at.unit >= a.units) return;
  float v[8];
  load_unit<T, PACKED>(static_cast<const T*>(a.x) + at.row * a.dim, at.e, a.dim, v);
  if (a.codes) {
    uint32_t code[2];
    const int s = mx_encode<kE4m3>(v, code);
    mx_store<kE4m3>(a.codes, a.scales, at.unit, code, s);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = gelu_f<T>(v[i]);
  store_unit<T, PACKED>(static_cast<T*>(a.y) + at.row * a.dim, at.e, a.dim, v);
}

// y = x * gelu'(kept): x is the gradient here.
template <typename T, bool PACKED>
__global__ __launch_bounds__(256) void gelu_backward_kernel(UnitArgs a) {
  const UnitPlace at(a);
  if (at.unit >= a.units) return;
  float g[8], v[8];
  load_unit<T, PACKED>(static_cast<const T*>(a.x) + at.row * a.dim, at.e, a.dim, g);
  mx_load<kE4m3>(a.codes, a.scales, at.unit, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] *= gelu_slope<T>(v[i]);
  store_unit<T, PACKED>(static_cast<T*>(a.y) + at.row * a.dim, at.e, a.dim, g);
}

int unit_args(const char* what, const void* x, void* y, const void* codes, const void* scales, int64_t rows,
              int64_t dim, int32_t type, UnitArgs& a, int64_t runs = 0) {
  JN_REQUIRE(known_type(type), kInvalidArgument, "%s: unknown element type %d", what, type);
  JN_REQUIRE(rows >= 1 && dim >= 1 && dim < (int64_t(1) << 31) && rows <= (int64_t(1) << 36) / mx_runs(dim),
             kInvalidArgument, "%s: needs rows and dim >= 1, dim < 2^31 and at most 2^36 runs, got %lld x %lld", what,
             (long long)rows, (long long)dim);
  JN_REQUIRE((codes == nullptr) == (scales == nullptr), kInvalidArgument, "%s: codes and scales come together", what);
  JN_REQUIRE(!codes || aligned16(codes), kInvalidArgument, "%s: codes must start on 16 bytes", what);
  a.x = x, a.y = y;
  a.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
  a.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  if (runs == 0) runs = mx_runs(dim);
  a.row_units = runs * 4, a.units = rows * a.row_units;
  const bool flat = dim == runs * kMxRun;
  a.rows = flat ? 1 : rows, a.dim = flat ? rows * dim : dim;
  return kOk;
}

// Whether the elements that a call reads and writes can move in packs of 16 bytes.
bool packed_rows(const UnitArgs& a, int32_t type) {
  return (!a.x || aligned16(a.x)) && (!a.y || aligned16(a.y)) && a.dim * type_bytes(type) % 16 == 0;
}

template <typename F>
int with_packs(bool packed, F f) {
  return packed ? f(std::true_type{}) : f(std::false_type{});
}
template <typename F>
int with_form(int32_t form, F f) {
  return form == kE4m3 ? f(std::integral_constant<int, kE4m3>{}) : f(std::integral_constant<int, kE2m1>{});
}

// A grid has fewer than 2^32 threads along an axis (what is asked beyond them is dropped
// without an error), so that more units go in several launches.
constexpr int64_t kLaunchUnits = int64_t(1) << 31;
template <typename F>
int launch_units(UnitArgs a, F launch) {
  for (; a.first < a.units; a.first += kLaunchUnits) {
    launch(dim3((unsigned)((std::min(kLaunchUnits, a.units - a.first) + 255) / 256)), a);
    JN_LAUNCH_CHECK();
  }
  return kOk;
}

}  // namespace

int launch_mx_quantize(const void* x, int64_t rows, int64_t dim, int32_t type, int32_t form, void* codes, void* scales,
                       hipStream_t s, int64_t runs) {
  UnitArgs a{};
  if (const int rc = unit_args("mx_quantize", x, nullptr, codes, scales, rows, dim, type, a, runs)) return rc;
  return with_type(type, [&](auto* t) -> int {
    return with_form(form, [&](auto f) -> int {
      return with_packs(packed_rows(a, type), [&](auto p) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        JN_PROFILE("mx_quantize_kernel", s);
        return launch_units(a, [&](dim3 grid, const UnitArgs& part) {
          hipLaunchKernelGGL((mx_quantize_kernel<T, f(), p()>), grid, dim3(256), 0, s, part);
        });
      });
    });
  });
}

}  // namespace jakal

using namespace jakal;

extern "C" {

int jn_mx_quantize(const void* x, int64_t rows, int64_t dim, int32_t type, int32_t format, void* codes, void* scales,
                   jn_stream_t stream) {
  JN_REQUIRE(x && codes && scales, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(known_form(format), kInvalidArgument, "mx_quantize: unknown format %d", format);
  return launch_mx_quantize(x, rows, dim, type, format, codes, scales, static_cast<hipStream_t>(stream));
}

int jn_mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t dim, int32_t format, int32_t type,
                     void* x, jn_stream_t stream) {
  JN_REQUIRE(x && codes && scales, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(known_form(format), kInvalidArgument, "mx_dequantize: unknown format %d", format);
  UnitArgs a{};
  if (const int rc = unit_args("mx_dequantize", nullptr, x, codes, scales, rows, dim, type, a)) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    return with_form(format, [&](auto f) -> int {
      return with_packs(packed_rows(a, type), [&](auto p) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        JN_PROFILE("mx_dequantize_kernel", s);
        return launch_units(a, [&](dim3 grid, const UnitArgs& part) {
          hipLaunchKernelGGL((mx_dequantize_kernel<T, f(), p()>), grid, dim3(256), 0, s, part);
        });
      });
    });
  });
}

int jn_gelu_forward(const void* x, int64_t rows, int64_t dim, int32_t type, void* y, void* codes, void* scales,
                    jn_stream_t stream) {
  JN_REQUIRE(x && y, kInvalidArgument, "null tensor pointer");
  UnitArgs a{};
  if (const int rc = unit_args("gelu", x, y, codes, scales, rows, dim, type, a)) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    return with_packs(packed_rows(a, type), [&](auto p) -> int {
      using T = std::remove_pointer_t<decltype(t)>;
      JN_PROFILE("gelu_forward_kernel", s);
      return launch_units(a, [&](dim3 grid, const UnitArgs& part) {
        hipLaunchKernelGGL((gelu_forward_kernel<T, p()>), grid, dim3(256), 0, s, part);
      });
    });
  });
}

int jn_gelu_backward(const void* codes, const void* scales, const void* grad_y, int64_t rows, int64_t dim,
                     int32_t type, void* grad_x, jn_stream_t stream) {
  JN_REQUIRE(codes && scales && grad_y && grad_x, kInvalidArgument, "null tensor pointer");
  UnitArgs a{};
  if (const int rc = unit_args("gelu backward", grad_y, grad_x, codes, scales, rows, dim, type, a)) return rc;
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    return with_packs(packed_rows(a, type), [&](auto p) -> int {
      using T = std::remove_pointer_t<decltype(t)>;
      JN_PROFILE("gelu_backward_kernel", s);
      return launch_units(a, [&](dim3 grid, const UnitArgs& part) {
        hipLaunchKernelGGL((gelu_backward_kernel<T, p()>), grid, dim3(256), 0, s, part);
      });
    });
  });
}

}  // extern "C"
