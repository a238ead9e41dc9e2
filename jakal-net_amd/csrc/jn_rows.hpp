// Element types and row reductions of the training-step operators (jn_norm.hip,
// jn_loss.hip, jn_clip.hip), which take fp32, bf16 and fp16 tensors and compute
// in fp32.
#pragma once

#include <type_traits>

#include "jn_common.hpp"

namespace jakal {

// Element type codes of the C ABI (JN_F32, JN_BF16, JN_F16 in jakal_net_hip.h).
constexpr int kTypeF32 = 0, kTypeBf16 = 1, kTypeF16 = 2;
typedef _Float16 f16_t;

inline bool known_type(int32_t t) { return t >= kTypeF32 && t <= kTypeF16; }
inline int type_bytes(int32_t t) { return t == kTypeF32 ? 4 : 2; }

// Calls f with a null pointer of the element type that a code names.
template <typename F>
int with_type(int32_t code, F f) {
  if (code == kTypeBf16) return f(static_cast<bf16_t*>(nullptr));
  if (code == kTypeF16) return f(static_cast<f16_t*>(nullptr));
  return f(static_cast<float*>(nullptr));
}

// One element of a tensor whose type is known at run time only (the branch is uniform).
__device__ __forceinline__ float load_any(const void* p, int64_t i, int code) {
  if (code == kTypeF32) return static_cast<const float*>(p)[i];
  if (code == kTypeBf16) return (float)static_cast<const bf16_t*>(p)[i];
  return (float)static_cast<const f16_t*>(p)[i];
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int code, float v) {
  if (code == kTypeF32) static_cast<float*>(p)[i] = v;
  else if (code == kTypeBf16) static_cast<bf16_t*>(p)[i] = (bf16_t)v;
  else static_cast<f16_t*>(p)[i] = (f16_t)v;
}

// W elements of T as one access: 16 or 8 bytes, or a single element.  STREAM:
// non-temporal, for data that the caches would not hold until its next use.
template <typename T, int W>
struct Raw {
  static_assert(W == 1 || W * sizeof(T) == 16 || W * sizeof(T) == 8, "a pack is one element, 8 or 16 bytes");
  using type = std::conditional_t<W == 1, T, std::conditional_t<W * sizeof(T) == 16, uint4, uint2>>;
  type bits;

  template <bool STREAM = false>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (STREAM && W * sizeof(T) == 16) bits = load_nt16(p);
    else if constexpr (STREAM && W * sizeof(T) == 8 && W > 1) bits = load_nt8(p);
    else bits = *reinterpret_cast<const type*>(p);
  }
  template <bool STREAM = false>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (STREAM && W * sizeof(T) == 16) store_nt16(p, bits);
    else if constexpr (STREAM && W * sizeof(T) == 8 && W > 1) store_nt8(p, bits);
    else *reinterpret_cast<type*>(p) = bits;
  }
  __device__ __forceinline__ void clear() { bits = type{}; }
  __device__ __forceinline__ void unpack(float* v) const {
    if constexpr (W == 1) {
      v[0] = (float)bits;
    } else {
      typedef T vec __attribute__((ext_vector_type(W)));
      const vec x = __builtin_bit_cast(vec, bits);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = (float)x[i];
    }
  }
  __device__ __forceinline__ void pack(const float* v) {
    if constexpr (W == 1) {
      bits = (T)v[0];
    } else {
      typedef T vec __attribute__((ext_vector_type(W)));
      vec x;
#pragma unroll
      for (int i = 0; i < W; ++i) x[i] = (T)v[i];
      bits = __builtin_bit_cast(type, x);
    }
  }
};

template <typename T, int W, bool STREAM = false>
__device__ __forceinline__ void store_raw(T* p, const float* v) {
  Raw<T, W> raw;
  raw.pack(v);
  raw.template store<STREAM>(p);
}

// The card's last-level cache: calls that move more than it holds stream.
constexpr int64_t kCacheBytes = 256LL << 20;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Sum over a workgroup of WAVES waves, the same in every thread (fixed order).
// `lds` holds WAVES floats and may be reused after the next barrier.
template <int WAVES>
__device__ __forceinline__ float group_sum(float v, float* lds) {
  v = wave_sum(v);
  if constexpr (WAVES == 1) return v;
  __syncthreads();  // earlier readers of lds are done
  if (lane_id() == 0) lds[wave_id()] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) s += lds[i];
  return s;
}

}  // namespace jakal
