// Microscaled numbers: runs of 32 elements of a row's last axis as short floats
// times one power of two (jn_mx.hip, jn_mx_product.hip).
//
//   e4m3: 8 bits, largest 448 = 1.75 * 2^8;  e2m1: 4 bits, largest 6 = 1.5 * 2^2
//   scale code s: 2^(s - 127), the smallest power of two >= 2^-126 that keeps the
//   run's largest magnitude within the format; 255 (the run is NaN) where the run
//   holds an infinity or a NaN
//   element code: x / 2^(s - 127) to the nearest value, ties to the even code
//
// In memory: codes row by row, each row padded with zeros to whole runs (e2m1 two a
// byte, the first in the low half), scales one byte a run.  The unit of work is
// eight elements a lane; four lanes of a quad make a run.
#pragma once

#include "jn_rows.hpp"

namespace jakal {

constexpr int kMxRun = 32;
constexpr int kE4m3 = 0, kE2m1 = 1;

inline bool known_form(int32_t f) { return f == kE4m3 || f == kE2m1; }
__host__ __device__ inline int64_t mx_runs(int64_t dim) { return (dim + kMxRun - 1) / kMxRun; }
// bytes of a row's codes
__host__ __device__ inline int64_t mx_pitch(int64_t dim, int form) {
  return mx_runs(dim) * (form == kE4m3 ? kMxRun : kMxRun / 2);
}

typedef float floatx2_t __attribute__((ext_vector_type(2)));

// The largest of four lanes of a quad, in each of them.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));         // lanes 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));      // lanes 2 3 0 1
}

// The scale code of a run by the bits of its largest magnitude (as integers, NaN
// lies above infinity and that above every number).
template <int FORM>
__device__ __forceinline__ int mx_scale_code(uint32_t bits) {
  constexpr int kTop = FORM == kE4m3 ? 8 : 2;
  constexpr uint32_t kSignificand = FORM == kE4m3 ? 0x600000u : 0x400000u;  // 1.75 and 1.5
  const int e = (int)(bits >> 23);
  const int s = e - kTop + ((bits & 0x7FFFFFu) > kSignificand ? 1 : 0);
  return e == 255 ? 255 : max(s, 1);
}

// 2^(s - 127); NaN for 255.
__device__ __forceinline__ float mx_scale(int s) {
  return __uint_as_float(s == 255 ? 0x7FC00000u : s == 0 ? 0x00400000u : (uint32_t)s << 23);
}

// Eight e2m1 codes of numbers within the format.
__device__ __forceinline__ uint32_t e2m1_word(const float (&v)[8]) {
  uint32_t a = 0;
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[0], v[1], 1.0f, 0);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[2], v[3], 1.0f, 1);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[4], v[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, v[6], v[7], 1.0f, 3);
}

// The codes of a lane's eight elements (e4m3: two words; e2m1: one) and its run's
// scale code.  |v| * 2^(127 - s) is within the format, so nothing saturates; the
// product is exact but where it falls below 2^-126, far under half the least code.
template <int FORM>
__device__ __forceinline__ int mx_encode(const float (&v)[8], uint32_t (&code)[2]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  const int s = mx_scale_code<FORM>(quad_max(most));
  const float inv = __uint_as_float((uint32_t)(254 - min(s, 253)) << 23);
  if constexpr (FORM == kE4m3) {
    int a = 0, b = 0;
    a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, a, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, a, true);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, b, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, b, true);
    code[0] = s == 255 ? 0x7F7F7F7Fu : (uint32_t)a;
    code[1] = s == 255 ? 0x7F7F7F7Fu : (uint32_t)b;
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i] * inv;
    code[0] = s == 255 ? 0u : e2m1_word(f);
    code[1] = 0;
  }
  return s;
}

// The values that eight codes stand for, before the scale.
template <int FORM>
__device__ __forceinline__ void mx_decode(const uint32_t (&code)[2], float (&v)[8]) {
  if constexpr (FORM == kE4m3) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const floatx2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[w], false);
      const floatx2_t b = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[w], true);
      v[4 * w] = a[0], v[4 * w + 1] = a[1], v[4 * w + 2] = b[0], v[4 * w + 3] = b[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // sign e e m: the magnitudes 0 .5 1 1.5 2 3 4 6
      const uint32_t c = code[0] >> (4 * i), e = (c >> 1) & 3u, m = c & 1u;
      const uint32_t size = e ? ((126u + e) << 23) | (m << 22) : m * 0x3F000000u;
      v[i] = __uint_as_float(size | ((c & 8u) << 28));
    }
  }
}

// A unit's codes in memory, and its run's scale.
template <int FORM>
__device__ __forceinline__ void mx_store(uint8_t* codes, uint8_t* scales, int64_t unit, const uint32_t (&code)[2],
                                         int s) {
  if constexpr (FORM == kE4m3) *reinterpret_cast<uint2*>(codes + unit * 8) = make_uint2(code[0], code[1]);
  else *reinterpret_cast<uint32_t*>(codes + unit * 4) = code[0];
  if ((unit & 3) == 0) scales[unit >> 2] = (uint8_t)s;
}
template <int FORM>
__device__ __forceinline__ void mx_load(const uint8_t* codes, const uint8_t* scales, int64_t unit, float (&v)[8]) {
  uint32_t code[2] = {0, 0};
  if constexpr (FORM == kE4m3) {
    const uint2 c = *reinterpret_cast<const uint2*>(codes + unit * 8);
    code[0] = c.x, code[1] = c.y;
  } else {
    code[0] = *reinterpret_cast<const uint32_t*>(codes + unit * 4);
  }
  const float scale = mx_scale(scales[unit >> 2]);
  mx_decode<FORM>(code, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= scale;
}

// Eight elements of a row from element e on, zeros past its end.  PACKED: rows
// start on 16 bytes and end on whole packs.
template <typename T, bool PACKED>
__device__ __forceinline__ void load_unit(const T* row, int64_t e, int64_t dim, float (&v)[8]) {
  if constexpr (PACKED) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      Raw<T, W> raw;
      if (e + i < dim) raw.load(row + e + i);
      else raw.clear();
      raw.unpack(v + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e + i < dim ? (float)row[e + i] : 0.f;
  }
}
template <typename T, bool PACKED>
__device__ __forceinline__ void store_unit(T* row, int64_t e, int64_t dim, const float (&v)[8]) {
  if constexpr (PACKED) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      if (e + i < dim) store_raw<T, W>(row + e + i, v + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (e + i < dim) row[e + i] = (T)v[i];
    }
  }
}

// jn_mx_quantize's launch, for the kernels that microscale an operand of their own:
// rows of `runs` runs where given, the surplus zeros.
int launch_mx_quantize(const void* x, int64_t rows, int64_t dim, int32_t type, int32_t form, void* codes, void* scales,
                       hipStream_t s, int64_t runs = 0);

}  // namespace jakal
