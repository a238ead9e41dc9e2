// Layer norm of rows, forward and backward, with the path scale and the state
// that a layer update carries beside it (jn_layer_norm_*).
//
//   v = scale * x,  m = mean(v),  r = 1 / sqrt(mean((v - m)^2) + eps),
//   h = (v - m) r,  y = h w + b;   state_out = tanh(scale * state)
//
//   g_w = g w;  dx = scale r (g_w - mean(g_w) - h mean(g_w h))
//   dw = sum over rows of g h,  db = sum over rows of g
//   dstate = scale (1 - tanh^2) g_state
//
// Or keeping c = x - p in e4m3 for the backward (jn_layer_norm_*_kept), p being the
// mean of x in 64 bits rounded to fp32: the forward is the same, h in the gradients
// is scale r times the kept c.  16 x 512 x 512 fp32 11.8 us forward (38 MB) and 12.0
// backward (38 MB, where reading x would be 50).  What is kept is centred so that its
// rounding is relative to h whatever the mean is.  A sum in 64 bits has 29 bits more than
// the numbers it adds: p, and with it the codes, is the same in any order of summing (the
// kernels' orders differ) unless the row cancels to within those bits (1e30, 1, -1e30, 3)
// or p falls on a border between two fp32 numbers; the codes are then those of a mean
// that differs in its last bits.
#include "../../include/jakal_net_hip.h"
#include "jn_internal.hpp"
#include "jn_mx.hpp"

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
  float* partial;   // [slabs][2][dim], or null: one workgroup has all sums, and writes dw and db
  void* dw;         // or null
  void* db;         // or null
  // the centred x in e4m3: written beside y, or read in x's place; or null
  uint8_t* codes;
  uint8_t* scales;
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

// ---- rows held in registers ---------------------------------------------------
// TH threads take a row: thread t of them the packs t, t + TH, ... of W elements
// (16 bytes; single elements where rows do not start on 16), NP packs and eight
// elements at most.  A row is read once, and its mean, centred squares and
// gradient sums come from registers; the next row's packs load while this one
// is reduced.  A workgroup of BLOCK threads holds several such groups, which
// step through the rows together (they share the barriers).
//
// The forward is bound by HBM once rows fill the chip (65,536 x 512: bf16 30 us,
// 4.4 TB/s of read and write; fp32 43 us, 6.2 TB/s), by one launch's latency below
// (64 x 512: 3.2 us); so is the backward (36 us, 5.7 TB/s; 78 us, 5.2 TB/s; 8,192 x
// 512 fp32 12 us).  Rows of single elements move 5.3 TB/s in fp32 and 3.1 in bf16
// (65,536 x 383 forward); 16-byte accesses at any element took the latter from 31
// to 71 us.
template <int W, int NP, int TH, int BLOCK>
struct RowGroup {
  static constexpr int kGroups = BLOCK / TH;
  static constexpr int kItems = W * NP;  // elements of a thread

  __device__ static int thread() { return TH == kWave ? lane_id() : (int)threadIdx.x % TH; }
  // of a group in the workgroup: uniform over a wave where groups are whole waves
  __device__ static int group() { return TH < kWave ? (int)threadIdx.x / TH : wave_id() / (TH / kWave); }
  __device__ static int element(int p) { return (p * TH + thread()) * W; }
};

// Sums of N values over each group of TH threads, the same in all of them.
template <int TH, int BLOCK, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float (*lds)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = row16_sum(v[i]);
    if constexpr (TH >= 32) v[i] += xor16_f(v[i]);
    if constexpr (TH >= 64) v[i] += xor32_f(v[i]);
  }
  if constexpr (TH > kWave) {
    constexpr int kWaves = TH / kWave;
    __syncthreads();  // the readers before are done
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[wave_id()][i] = v[i];
    }
    __syncthreads();
    const int first = wave_id() / kWaves * kWaves;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) v[i] += lds[first + k][i];
    }
  }
}

template <typename T, int W, int NP, typename G>
__device__ __forceinline__ void load_row(const void* base, int64_t row, const NormArgs& a, Raw<T, W> (&raw)[NP]) {
  const T* p = static_cast<const T*>(base) + row * a.dim;
  if (row >= a.rows) {
#pragma unroll
    for (int i = 0; i < NP; ++i) raw[i].clear();
    return;
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int e = G::element(i);
    if (e < a.dim) raw[i].load(p + e);
    else raw[i].clear();
  }
}

// W elements of a row kept in e4m3, and their run's scale.
template <int W>
struct KeptPack {
  std::conditional_t<W == 1, uint8_t, std::conditional_t<W == 4, uint32_t, uint2>> code;
  uint8_t scale;

  __device__ __forceinline__ void clear() { code = {}, scale = 127; }
  __device__ __forceinline__ void unpack(float* v) const {
    const float f = mx_scale(scale);
    if constexpr (W == 1) {
      v[0] = __builtin_amdgcn_cvt_f32_fp8((int)code, 0) * f;
    } else {
      uint32_t words[2] = {0, 0};
      if constexpr (W == 4) words[0] = code;
      else words[0] = code.x, words[1] = code.y;
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const floatx2_t x = i % 4 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)words[i / 4], true)
                                  : __builtin_amdgcn_cvt_pk_f32_fp8((int)words[i / 4], false);
        v[i] = x[0] * f, v[i + 1] = x[1] * f;
      }
    }
  }
};

template <typename T, int W, int NP, typename G>
__device__ __forceinline__ void load_row(const NormArgs& a, int64_t row, KeptPack<W> (&kept)[NP]) {
  const uint8_t* codes = a.codes + row * mx_pitch(a.dim, kE4m3);
  const uint8_t* scales = a.scales + row * mx_runs(a.dim);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int e = G::element(i);
    if (row < a.rows && e < a.dim) {
      kept[i].code = *reinterpret_cast<const decltype(kept[i].code)*>(codes + e);
      kept[i].scale = scales[e / kMxRun];
    } else {
      kept[i].clear();
    }
  }
}
template <typename T, int W, int NP, typename G>
__device__ __forceinline__ void load_row(const NormArgs& a, int64_t row, Raw<T, W> (&raw)[NP]) {
  load_row<T, W, NP, G>(a.x, row, a, raw);
}

// A value from another lane, both its words moved alike.
template <typename F>
__device__ __forceinline__ double moved(double v, F move) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = (uint32_t)move((int)(uint32_t)u), hi = (uint32_t)move((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, lo | hi << 32);
}
template <int CTRL>
__device__ __forceinline__ double dpp_64(double v) {
  return moved(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, true); });
}

// The sum of a value over each group of TH threads in 64 bits, in all of them.
template <int TH, int BLOCK>
__device__ __forceinline__ double group_sum_64(double v, double* lds) {
  v += dpp_64<0xB1>(v), v += dpp_64<0x4E>(v), v += dpp_64<0x141>(v), v += dpp_64<0x140>(v);  // sixteen lanes
  if constexpr (TH >= 32) v += moved(v, [](int x) { return xor16_i(x); });
  if constexpr (TH >= 64) v += moved(v, [](int x) { return xor32_i(x); });
  if constexpr (TH > kWave) {
    constexpr int kWaves = TH / kWave;
    __syncthreads();  // the readers before are done
    if (lane_id() == 0) lds[wave_id()] = v;
    __syncthreads();
    const int first = wave_id() / kWaves * kWaves;
    v = 0.0;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) v += lds[first + k];
  }
  return v;
}

// Keeps a row, centred, in e4m3: the largest of a run's elements over the 32 / W lanes
// that hold it (two packs of sixteen lanes where rows of single elements have no more).
template <int W, int NP, int TH, int BLOCK, typename G>
__device__ __forceinline__ void keep_row(const NormArgs& a, int64_t row, const float* x, double* lds) {
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < W * NP; ++i) sum += x[i];  // (zeros past the row's end)
  const float p = (float)(group_sum_64<TH, BLOCK>(sum, lds) / (double)a.dim);
  float v[W * NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
#pragma unroll
    for (int j = i * W; j < i * W + W; ++j) v[j] = G::element(i) < a.dim ? x[j] - p : 0.f;
  }
  uint32_t most[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    most[i] = 0;
#pragma unroll
    for (int j = 0; j < W; ++j) most[i] = max(most[i], __float_as_uint(v[i * W + j]) & 0x7FFFFFFFu);
  }
  constexpr bool kPairs = W == 1 && TH == 16;
  static_assert(!kPairs || NP % 2 == 0, "a run is two packs");
  if constexpr (kPairs) {
#pragma unroll
    for (int i = 0; i < NP; i += 2) most[i] = most[i + 1] = max(most[i], most[i + 1]);
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    most[i] = quad_max(most[i]);
    if constexpr (W <= 4)  // eight lanes
      most[i] = max(most[i], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most[i], 0x141, 0xF, 0xF, true));
    if constexpr (W == 1) {  // sixteen, and 32
      most[i] = max(most[i], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most[i], 0x140, 0xF, 0xF, true));
      if constexpr (!kPairs) most[i] = max(most[i], (uint32_t)xor16_i((int)most[i]));
    }
  }
  if (row >= a.rows) return;
  const int64_t pitch = mx_pitch(a.dim, kE4m3);
  uint8_t* codes = a.codes + row * pitch;
  uint8_t* scales = a.scales + row * mx_runs(a.dim);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int e = G::element(i);
    if (e >= pitch) continue;
    const int s = mx_scale_code<kE4m3>(most[i]);
    const float inv = __uint_as_float((uint32_t)(254 - min(s, 253)) << 23);
    uint32_t words[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < W; j += 2) {
      const float x = v[i * W + j] * inv, y = W > 1 ? v[i * W + (W > 1 ? j + 1 : j)] * inv : 0.f;
      words[j / 4] = j % 4 ? __builtin_amdgcn_cvt_pk_fp8_f32(x, y, (int)words[j / 4], true)
                           : __builtin_amdgcn_cvt_pk_fp8_f32(x, y, (int)words[j / 4], false);
    }
    if (s == 255) words[0] = words[1] = 0x7F7F7F7Fu;
    if constexpr (W == 1) codes[e] = (uint8_t)words[0];
    else if constexpr (W == 4) *reinterpret_cast<uint32_t*>(codes + e) = words[0];
    else *reinterpret_cast<uint2*>(codes + e) = make_uint2(words[0], words[1]);
    if (e % kMxRun == 0) scales[e / kMxRun] = (uint8_t)s;
  }
}

// The same for rows of any width: a workgroup a row.
template <typename T>
__global__ __launch_bounds__(256) void norm_keep_any_kernel(NormArgs a) {
  __shared__ double lds[4];
  const int64_t units = mx_runs(a.dim) * 4;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.dim;
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < a.dim; i += 256) sum += (double)(float)x[i];
    const float p = (float)(group_sum_64<256, 256>(sum, lds) / (double)a.dim);
    for (int64_t u = threadIdx.x; u < units; u += 256) {  // whole quads
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = u * 8 + j < a.dim ? (float)x[u * 8 + j] - p : 0.f;
      uint32_t code[2];
      const int s = mx_encode<kE4m3>(v, code);
      mx_store<kE4m3>(a.codes, a.scales, row * units + u, code, s);
    }
  }
}

// h of element i of a row: from x, or from what was kept of it.
template <typename T, bool KEPT>
struct RowReader {
  const T* x;
  const uint8_t* codes;
  const uint8_t* scales;
  float scale, m, r;

  __device__ RowReader(const NormArgs& a, int64_t row) {
    if constexpr (KEPT) codes = a.codes + row * mx_pitch(a.dim, kE4m3), scales = a.scales + row * mx_runs(a.dim);
    else x = static_cast<const T*>(a.x) + row * a.dim;
    scale = a.scale, m = a.stats[2 * row], r = a.stats[2 * row + 1];
  }
  __device__ __forceinline__ float operator[](int64_t i) const {
    if constexpr (KEPT) {
      return scale * (__builtin_amdgcn_cvt_f32_fp8((int)codes[i], 0) * mx_scale(scales[i / kMxRun])) * r;
    } else {
      return (scale * (float)x[i] - m) * r;
    }
  }
};

template <typename T, int W, int NP, typename G>
__device__ __forceinline__ void load_params(const void* base, int type, int64_t dim, float none,
                                            float (&v)[W * NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int e = G::element(i);
#pragma unroll
    for (int j = 0; j < W; ++j) v[i * W + j] = none;
    if (!base || e >= dim) continue;
    if (sizeof(T) != 4 && type != kTypeF32) {
      Raw<T, W> raw;
      raw.load(static_cast<const T*>(base) + e);
      raw.unpack(v + i * W);
    } else {
      const float* p = static_cast<const float*>(base) + e;
      if constexpr (W == 1) {
        v[i] = p[0];
      } else {
#pragma unroll
        for (int j = 0; j < W; j += 4) {
          Raw<float, 4> raw;
          raw.load(p + j);
          raw.unpack(v + i * W + j);
        }
      }
    }
  }
}

template <typename T, int W, int NP, int TH, int BLOCK, bool KEEP>
__global__ __launch_bounds__(BLOCK) void norm_forward_kernel(NormArgs a) {
  using G = RowGroup<W, NP, TH, BLOCK>;
  __shared__ float lds[BLOCK / kWave][1];
  __shared__ double lds64[KEEP ? BLOCK / kWave : 1];
  const int64_t step = (int64_t)gridDim.x * G::kGroups;
  int64_t base = (int64_t)blockIdx.x * G::kGroups;
  const int group = G::group();
  const float n = (float)a.dim;
  Raw<T, W> next[NP];
  load_row<T, W, NP, G>(a.x, base + group, a, next);
  float w[G::kItems], b[G::kItems];
  load_params<T, W, NP, G>(a.w, a.param_type, a.dim, 1.0f, w);
  load_params<T, W, NP, G>(a.b, a.param_type, a.dim, 0.0f, b);
  for (; base < a.rows; base += step) {
    const int64_t row = base + group;
    float v[G::kItems];
#pragma unroll
    for (int i = 0; i < NP; ++i) next[i].unpack(v + i * W);
    if (base + step < a.rows) load_row<T, W, NP, G>(a.x, row + step, a, next);
    if constexpr (KEEP) keep_row<W, NP, TH, BLOCK, G>(a, row, v, lds64);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < G::kItems; ++i) {
      v[i] *= a.scale;
      s[0] += v[i];
    }
    group_sums<TH, BLOCK>(s, lds);
    const float m = s[0] / n;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (G::element(i) >= a.dim) continue;  // (the clears there are not elements)
#pragma unroll
      for (int j = 0; j < W; ++j) {
        v[i * W + j] -= m;
        s[0] += v[i * W + j] * v[i * W + j];
      }
    }
    group_sums<TH, BLOCK>(s, lds);
    const float r = 1.0f / sqrtf(s[0] / n + a.eps);
    if (row >= a.rows) continue;
    T* y = static_cast<T*>(a.y) + row * a.dim;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (G::element(i) >= a.dim) continue;
#pragma unroll
      for (int j = 0; j < W; ++j) v[i * W + j] = v[i * W + j] * r * w[i * W + j] + b[i * W + j];
      store_raw<T, W>(y + G::element(i), v + i * W);
    }
    if (a.stats && G::thread() == 0) {
      a.stats[2 * row] = m;
      a.stats[2 * row + 1] = r;
    }
  }
  if (a.state) {
    for (int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x; i < a.rows; i += (int64_t)gridDim.x * BLOCK)
      state_forward(a, i);
  }
}

// Each thread also keeps its own columns' sums in registers; the groups of a
// workgroup join in LDS at the end.
template <typename T, int W, int NP, int TH, int BLOCK, bool KEPT>
__global__ __launch_bounds__(BLOCK) void norm_backward_kernel(NormArgs a) {
  using G = RowGroup<W, NP, TH, BLOCK>;
  __shared__ float lds[BLOCK / kWave][2];
  extern __shared__ float sums[];  // [kGroups][dim], at most 16 KB
  const int64_t step = (int64_t)gridDim.x * G::kGroups;
  const int group = G::group();
  const float n = (float)a.dim;
  float dw[G::kItems], db[G::kItems];
#pragma unroll
  for (int i = 0; i < G::kItems; ++i) dw[i] = db[i] = 0.f;
  if (a.dx || a.dw || a.db) {
    int64_t base = (int64_t)blockIdx.x * G::kGroups;
    std::conditional_t<KEPT, KeptPack<W>, Raw<T, W>> next_x[NP];
    Raw<T, W> next_g[NP];
    load_row<T, W, NP, G>(a, base + group, next_x);
    load_row<T, W, NP, G>(a.g, base + group, a, next_g);
    float w[G::kItems];
    load_params<T, W, NP, G>(a.w, a.param_type, a.dim, 1.0f, w);
    for (; base < a.rows; base += step) {
      const int64_t row = base + group;
      const bool live = row < a.rows;  // (a dead row is all zeros)
      const float m = live ? a.stats[2 * row] : 0.f, r = live ? a.stats[2 * row + 1] : 0.f;
      float h[G::kItems], g[G::kItems];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        next_x[i].unpack(h + i * W);
        next_g[i].unpack(g + i * W);
      }
      if (base + step < a.rows) {
        load_row<T, W, NP, G>(a, row + step, next_x);
        load_row<T, W, NP, G>(a.g, row + step, a, next_g);
      }
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (G::element(i) >= a.dim) continue;
#pragma unroll
        for (int j = i * W; j < i * W + W; ++j) {
          h[j] = KEPT ? a.scale * h[j] * r : (a.scale * h[j] - m) * r;
          dw[j] += g[j] * h[j];
          db[j] += g[j];
          g[j] *= w[j];
          s[0] += g[j];
          s[1] += g[j] * h[j];
        }
      }
      if (!a.dx) continue;
      group_sums<TH, BLOCK>(s, lds);
      const float s1 = s[0] / n, s2 = s[1] / n, sr = a.scale * r;
      T* dx = static_cast<T*>(a.dx) + row * a.dim;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (!live || G::element(i) >= a.dim) continue;
#pragma unroll
        for (int j = i * W; j < i * W + W; ++j) h[j] = sr * (g[j] - s1 - h[j] * s2);
        store_raw<T, W>(dx + G::element(i), h + i * W);
      }
    }
  }
  if (a.dstate) {
    for (int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x; i < a.rows; i += (int64_t)gridDim.x * BLOCK)
      state_backward(a, i);
  }
  if (!a.dw && !a.db) return;
  const auto put = [&](int k, int c, float v) {
    if (a.partial) a.partial[((int64_t)blockIdx.x * 2 + k) * a.dim + c] = v;
    else if (k ? a.db : a.dw) store_any(k ? a.db : a.dw, c, a.param_type, v);
  };
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k) __syncthreads();  // the sums before are read
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int e = G::element(i);
      if (e >= a.dim) continue;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float v = k ? db[i * W + j] : dw[i * W + j];
        if (G::kGroups == 1) put(k, e + j, v);
        else sums[group * (int)a.dim + e + j] = v;
      }
    }
    if (G::kGroups == 1) continue;
    __syncthreads();
    for (int c = threadIdx.x; c < (int)a.dim; c += BLOCK) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < G::kGroups; ++i) s += sums[i * (int)a.dim + c];
      put(k, c, s);
    }
  }
}

// Rows of any width and alignment: a workgroup a row, three passes over it, two of
// them from L2 (fp32, forward and input gradient: 1,024 x 16,384 74 and 74 us,
// 2,048 x 16,384 116 and 125, 512 x 33,000 106 and 130; the column sums take 22,
// 51 and 28 more, the join 8 to 14).
constexpr int kAnyThreads = 256;
constexpr int kAnyWaves = kAnyThreads / kWave;

// The sum of term(i) over a row by a workgroup, the same in every thread.  A
// thread adds 256 terms in fp32 and those sums in 64 bits: a row of 2^28 gives
// it 2^20 terms, whose sum in fp32 alone drops digits of every term (of a constant
// 0.1 the mean of 2^26 came out 150 times as far off as runs of 256 may be).  Eight
// loads in flight: one at a time the three forwards took 100, 116 and 163 us.
constexpr int64_t kRun = 256 * kAnyThreads;  // elements
template <typename F>
__device__ __forceinline__ float row_sum(int64_t dim, float* lds, F term) {
  double s = 0.0;
  for (int64_t first = 0; first < dim; first += kRun) {
    const int64_t end = min(dim, first + kRun);
    float run = 0.f;
#pragma unroll 8
    for (int64_t i = first + threadIdx.x; i < end; i += kAnyThreads) run += term(i);
    s += run;
  }
  return group_sum<kAnyWaves>((float)s, lds);
}

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void norm_forward_any_kernel(NormArgs a) {
  __shared__ float lds[kAnyWaves];
  const float n = (float)a.dim;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.dim;
    T* y = static_cast<T*>(a.y) + row * a.dim;
    const float m = row_sum(a.dim, lds, [&](int64_t i) { return a.scale * (float)x[i]; }) / n;
    const float var = row_sum(a.dim, lds, [&](int64_t i) {
      const float c = a.scale * (float)x[i] - m;
      return c * c;
    }) / n;
    const float r = 1.0f / sqrtf(var + a.eps);
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

template <typename T, bool KEPT>
__global__ __launch_bounds__(kAnyThreads) void norm_backward_any_kernel(NormArgs a) {
  __shared__ float lds[kAnyWaves];
  const float n = (float)a.dim;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (a.dstate && threadIdx.x == 0) state_backward(a, row);
    if (!a.dx) continue;
    const RowReader<T, KEPT> h(a, row);
    const T* g = static_cast<const T*>(a.g) + row * a.dim;
    T* dx = static_cast<T*>(a.dx) + row * a.dim;
    double d1 = 0.0, d2 = 0.0;
    for (int64_t first = 0; first < a.dim; first += kRun) {
      const int64_t end = min(a.dim, first + kRun);
      float run1 = 0.f, run2 = 0.f;
      for (int64_t i = first + threadIdx.x; i < end; i += kAnyThreads) {
        const float gw = (float)g[i] * param(a.w, i, a.param_type, 1.0f);
        run1 += gw;
        run2 += gw * h[i];
      }
      d1 += run1, d2 += run2;
    }
    const float s1 = group_sum<kAnyWaves>((float)d1, lds) / n;
    const float s2 = group_sum<kAnyWaves>((float)d2, lds) / n;
    const float sr = a.scale * h.r;
    for (int64_t i = threadIdx.x; i < a.dim; i += kAnyThreads) {
      const float gw = (float)g[i] * param(a.w, i, a.param_type, 1.0f);
      dx[i] = (T)(sr * (gw - s1 - h[i] * s2));
    }
  }
}

// Partial column sums of g h and g: a workgroup takes 64 columns of a slab of
// rows, its four waves every fourth row.
template <typename T, bool KEPT>
__global__ __launch_bounds__(kAnyThreads) void norm_columns_any_kernel(NormArgs a, int64_t slab_rows) {
  __shared__ float lds[2][kAnyWaves][kWave];
  const int64_t c = (int64_t)blockIdx.x * kWave + lane_id();
  const int64_t r0 = (int64_t)blockIdx.y * slab_rows;
  const int64_t r1 = r0 + slab_rows < a.rows ? r0 + slab_rows : a.rows;
  float sw = 0.f, sb = 0.f;
  if (c < a.dim) {
    for (int64_t row = r0 + wave_id(); row < r1; row += kAnyWaves) {
      const float g = (float)static_cast<const T*>(a.g)[row * a.dim + c];
      sw += g * RowReader<T, KEPT>(a, row)[c];
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

// The partial sums of all workgroups or slabs: 16 columns a workgroup at a time,
// each by 64 threads that take every 64th partial (512 x 1024 sums in 3.9 us).
// A launch has fewer than 2^32 threads along an axis, which 2^25 columns of dw
// and db would reach in workgroups of their own, so that those step.
constexpr int kFinishColumns = 16, kFinishLanes = 64;
constexpr int64_t kFinishGroups = 1 << 16;
__global__ __launch_bounds__(kFinishColumns* kFinishLanes) void norm_columns_finish_kernel(NormArgs a, int parts) {
  __shared__ float lds[kFinishLanes][kFinishColumns + 1];
  const int col = threadIdx.x % kFinishColumns, lane = threadIdx.x / kFinishColumns;
  for (int64_t first = (int64_t)blockIdx.x * kFinishColumns; first < 2 * a.dim;
       first += (int64_t)gridDim.x * kFinishColumns) {
    const int64_t c = first + col;  // of dw's columns and then db's
    float s = 0.f;
    if (c < 2 * a.dim) {
#pragma unroll 4
      for (int p = lane; p < parts; p += kFinishLanes) s += a.partial[(int64_t)p * 2 * a.dim + c];
    }
    lds[lane][col] = s;
    for (int step = kFinishLanes / 2; step > 0; step /= 2) {
      __syncthreads();
      if (lane < step) lds[lane][col] += lds[lane + step][col];
    }
    if (lane == 0 && c < 2 * a.dim) {
      void* out = c < a.dim ? a.dw : a.db;
      if (out) store_any(out, c < a.dim ? c : c - a.dim, a.param_type, lds[0][col]);
    }
    __syncthreads();
  }
}

// ---- which kernel ---------------------------------------------------------------
// The register kernels' shapes: packs of 16 bytes where every row and parameter
// starts on 16, else single elements; eight elements a thread (of sixteen the
// backward has the registers for three waves a SIMD: 16,384 x 1,536 bf16 took
// 59 us so, 39 now), by as few threads as hold the row, sixteen at least (a wave
// for every row took 30 us for the backward of 65,536 x 64 fp32, sixteen lanes
// take 11).  Rows that 1024 threads do not hold take the kernels that pass over
// memory.
struct RowShape {
  int width, items, threads;  // W, W * NP, TH; threads = 0: none fits
};

RowShape row_shape(int64_t dim, bool aligned, int elem_bytes) {
  const int w = aligned ? 16 / elem_bytes : 1;
  if (dim > 8 * 1024) return {w, 0, 0};
  int threads = 16;
  while (dim > 8 * threads) threads *= 2;
  return {w, w <= 4 && dim <= 4 * threads ? 4 : 8, threads};
}

template <int N>
using Int = std::integral_constant<int, N>;

// Calls f(W, NP, TH) with a shape's numbers as constants.
template <int V, typename F>
int with_shape(const RowShape& s, F f) {
  const auto packed = [&](auto width) -> int {
    constexpr int W = decltype(width)::value;
    if constexpr (W <= 4) {
      if (s.items == 4) return f(width, Int<4 / W>{}, Int<16>{});  // (up to 64 elements)
    }
    switch (s.threads) {
      case 16:
        return f(width, Int<8 / W>{}, Int<16>{});
      case 32:
        return f(width, Int<8 / W>{}, Int<32>{});
      case 64:
        return f(width, Int<8 / W>{}, Int<64>{});
      case 128:
        return f(width, Int<8 / W>{}, Int<128>{});
      case 256:
        return f(width, Int<8 / W>{}, Int<256>{});
      case 512:
        return f(width, Int<8 / W>{}, Int<512>{});
      default:
        return f(width, Int<8 / W>{}, Int<1024>{});
    }
  };
  return s.width == 1 ? packed(Int<1>{}) : packed(Int<V>{});
}

// Threads of a workgroup of the backward, and its workgroups, each of which
// leaves one row of partial sums.  65,536 x 512 bf16 with the join: 512 threads
// and up to 512 workgroups 42 us, 1024 and 512 46, 1024 and 256 43, 256 and
// 512 59, 256 and 1024 44; 8,192 x 512 fp32: 15.9, 19.2, 16.9, 15.7 and 16.4;
// 4,593 x 383: 13.2, 15.4, 12.8, 13.6 and 14.5.  Fewer rows take 256, so that
// the workgroups fill the CUs.
constexpr int64_t kMaxParts = 512;
constexpr int64_t kManyRows = 2048;
constexpr int64_t kFewSteps = 2;

// A workgroup that has all rows in two steps needs no partial sums and no second
// launch (fp32, captured, one launch against two: one step 8 x 512 3.9 against 6.0
// us, 32 x 64 3.3 and 5.0; two steps 16 x 512 4.8 and 6.1, 2 x 4,096 6.0 and 7.8;
// four 32 x 512 6.6 and 6.2, 16 x 1,024 7.7 and 6.6, 4 x 4,096 8.2 and 7.8).  The
// second launch costs the host 4 us.
bool one_workgroup(const RowShape& s, int64_t rows) { return rows <= kFewSteps * std::max(512 / s.threads, 1); }

struct BackwardGrid {
  int block;
  int64_t groups;
};

BackwardGrid backward_grid(const RowShape& s, int64_t rows, bool columns) {
  const bool one = columns && one_workgroup(s, rows);
  const int block = std::max(s.threads, one || rows >= kManyRows ? 512 : 256);
  const int64_t per = block / s.threads;
  return {block, one ? 1 : std::min((rows + per - 1) / per, kMaxParts)};
}

// Row slabs of the column sums of wide rows.
constexpr int64_t kSlabs = 64;
int64_t slab_count(int64_t rows) { return std::min<int64_t>(kSlabs, (rows + 15) / 16); }

// Rows of partial sums that a backward with parameter gradients leaves: a slab's
// or a workgroup's each (the shape's threads go by the width alone).  A single
// workgroup leaves none, and is given one.
int64_t part_count(int64_t rows, int64_t dim) {
  const RowShape shape = row_shape(dim, false, sizeof(float));
  return shape.threads ? backward_grid(shape, rows, true).groups : slab_count(rows);
}

// Workgroups of the forward: eight of four waves a CU.
constexpr int64_t kForwardGroups = 2048;

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

template <typename T>
bool aligned_rows(const NormArgs& a) {
  if (a.dim % (16 / sizeof(T)) != 0) return false;
  for (const void* p : {a.x, static_cast<const void*>(a.y), a.g, static_cast<const void*>(a.dx), a.w, a.b}) {
    if (!aligned16(p)) return false;
  }
  return true;
}

template <typename T, bool KEEP>
int launch_norm_forward(const NormArgs& a, hipStream_t s) {
  const bool aligned = aligned_rows<T>(a);
  const RowShape shape = row_shape(a.dim, aligned, sizeof(T));
  if (!shape.threads) {
    {
      JN_PROFILE("norm_forward_any_kernel", s);
      hipLaunchKernelGGL(norm_forward_any_kernel<T>, dim3((unsigned)row_groups(a.rows)), dim3(kAnyThreads), 0, s, a);
      JN_LAUNCH_CHECK();
    }
    if constexpr (KEEP) {
      JN_PROFILE("norm_keep_any_kernel", s);
      hipLaunchKernelGGL(norm_keep_any_kernel<T>, dim3((unsigned)row_groups(a.rows)), dim3(256), 0, s, a);
      JN_LAUNCH_CHECK();
    }
    return kOk;
  }
  return with_shape<16 / sizeof(T)>(shape, [&](auto width, auto packs, auto threads) -> int {
    constexpr int W = decltype(width)::value, NP = decltype(packs)::value, TH = decltype(threads)::value;
    constexpr int kBlock = TH > 256 ? TH : 256, per = kBlock / TH;
    const unsigned grid = (unsigned)std::min<int64_t>((a.rows + per - 1) / per, kForwardGroups);
    JN_PROFILE("norm_forward_kernel", s);
    hipLaunchKernelGGL((norm_forward_kernel<T, W, NP, TH, kBlock, KEEP>), dim3(grid), dim3(kBlock), 0, s, a);
    JN_LAUNCH_CHECK();
    return kOk;
  });
}

int launch_columns_finish(const NormArgs& a, int64_t parts, hipStream_t s) {
  const int64_t groups = std::min((2 * a.dim + kFinishColumns - 1) / kFinishColumns, kFinishGroups);
  JN_PROFILE("norm_columns_finish_kernel", s);
  hipLaunchKernelGGL(norm_columns_finish_kernel, dim3((unsigned)groups), dim3(kFinishColumns * kFinishLanes), 0, s, a,
                     (int)parts);
  JN_LAUNCH_CHECK();
  return kOk;
}

template <typename T, bool KEPT>
int launch_norm_backward(NormArgs a, hipStream_t s) {
  const bool columns = a.dw || a.db;
  if (!columns && !a.dx && !a.dstate) return kOk;
  const bool aligned = aligned_rows<T>(a);
  const RowShape shape = row_shape(a.dim, aligned, sizeof(T));
  if (!shape.threads) {
    if (a.dx || a.dstate) {
      JN_PROFILE("norm_backward_any_kernel", s);
      hipLaunchKernelGGL((norm_backward_any_kernel<T, KEPT>), dim3((unsigned)row_groups(a.rows)), dim3(kAnyThreads), 0, s,
                         a);
      JN_LAUNCH_CHECK();
    }
    if (!columns) return kOk;
    const int64_t slabs = slab_count(a.rows);
    {
      JN_PROFILE("norm_columns_any_kernel", s);
      hipLaunchKernelGGL((norm_columns_any_kernel<T, KEPT>), dim3((unsigned)((a.dim + kWave - 1) / kWave), (unsigned)slabs),
                         dim3(kAnyThreads), 0, s, a, (a.rows + slabs - 1) / slabs);
      JN_LAUNCH_CHECK();
    }
    return launch_columns_finish(a, slabs, s);
  }
  const BackwardGrid grid = backward_grid(shape, a.rows, columns);
  if (!columns || grid.groups == 1) a.partial = nullptr;
  const int rc = with_shape<16 / sizeof(T)>(shape, [&](auto width, auto packs, auto threads) -> int {
    constexpr int W = decltype(width)::value, NP = decltype(packs)::value, TH = decltype(threads)::value;
    const auto run = [&](auto block) -> int {
      constexpr int kBlock = decltype(block)::value;
      const size_t lds = columns && kBlock > TH ? (size_t)(kBlock / TH) * a.dim * sizeof(float) : 0;
      JN_PROFILE("norm_backward_kernel", s);
      hipLaunchKernelGGL((norm_backward_kernel<T, W, NP, TH, kBlock, KEPT>), dim3((unsigned)grid.groups), dim3(kBlock),
                         lds, s, a);
      JN_LAUNCH_CHECK();
      return kOk;
    };
    if constexpr (TH >= 512) return run(Int<TH>{});
    else return grid.block == 512 ? run(Int<512>{}) : run(Int<256>{});
  });
  if (rc || !a.partial) return rc;
  return launch_columns_finish(a, grid.groups, s);
}

}  // namespace
}  // namespace jakal

using namespace jakal;

namespace {

int forward(const void* state, const void* x, const void* weight, const void* bias, int64_t rows, int64_t dim,
            float scale, float eps, int32_t type, int32_t state_type, int32_t param_type, void* state_out, void* y,
            float* stats, bool keep, void* codes, void* scales, jn_stream_t stream) {
  NormArgs a{};
  a.x = x, a.w = weight, a.b = bias, a.state = state, a.rows = rows, a.dim = dim, a.scale = scale, a.eps = eps;
  a.state_type = state_type, a.param_type = param_type, a.y = y, a.state_out = state_out, a.stats = stats;
  a.codes = static_cast<uint8_t*>(codes), a.scales = static_cast<uint8_t*>(scales);
  if (const int rc = check_norm(a, type, state_type, param_type)) return rc;
  JN_REQUIRE(eps >= 0.0f, kInvalidArgument, "layer norm: eps must not be negative");
  if (rows == 0) return kOk;
  JN_REQUIRE(x && y && (!state || state_out), kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(!keep || (codes && scales && aligned16(codes)), kInvalidArgument,
             "layer norm: codes and scales to keep x in, the codes on a 16-byte address");
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    return keep ? launch_norm_forward<T, true>(a, s) : launch_norm_forward<T, false>(a, s);
  });
}

int backward(const void* state, const void* x, const void* weight, const float* stats, const void* grad_state_out,
             const void* grad_y, int64_t rows, int64_t dim, float scale, int32_t type, int32_t state_type,
             int32_t param_type, void* grad_state, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
             size_t workspace_bytes, bool kept, const void* codes, const void* scales, jn_stream_t stream) {
  NormArgs a{};
  a.x = x, a.w = weight, a.state = state, a.rows = rows, a.dim = dim, a.scale = scale;
  a.state_type = state_type, a.param_type = param_type, a.stats = const_cast<float*>(stats);
  a.g = grad_y, a.g_state = grad_state_out, a.dx = grad_x, a.dstate = grad_state;
  a.partial = static_cast<float*>(workspace), a.dw = grad_weight, a.db = grad_bias;
  a.codes = static_cast<uint8_t*>(const_cast<void*>(codes)), a.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  if (const int rc = check_norm(a, type, state_type, param_type)) return rc;
  JN_REQUIRE(rows >= 1, kInvalidArgument, "layer norm backward needs at least one row");
  const bool columns = grad_weight || grad_bias;
  JN_REQUIRE(!grad_state || (state && grad_state_out), kInvalidArgument, "null tensor pointer");
  JN_REQUIRE((!grad_x && !columns) || ((kept ? codes && scales : x != nullptr) && stats && grad_y), kInvalidArgument,
             "null tensor pointer");
  JN_REQUIRE(!kept || aligned16(codes), kInvalidArgument, "layer norm: codes must start on 16 bytes");
  const size_t need = columns ? jn_layer_norm_backward_workspace_bytes(rows, dim) : 0;
  JN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), kWorkspaceTooSmall,
             "layer norm backward needs %zu workspace bytes, got %zu", need, workspace_bytes);
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    return kept ? launch_norm_backward<T, true>(a, s) : launch_norm_backward<T, false>(a, s);
  });
}

}  // namespace

extern "C" {

int jn_layer_norm_forward(const void* state, const void* x, const void* weight, const void* bias, int64_t rows,
                          int64_t dim, float scale, float eps, int32_t type, int32_t state_type, int32_t param_type,
                          void* state_out, void* y, float* stats, jn_stream_t stream) {
  return forward(state, x, weight, bias, rows, dim, scale, eps, type, state_type, param_type, state_out, y, stats,
                 false, nullptr, nullptr, stream);
}

int jn_layer_norm_forward_kept(const void* state, const void* x, const void* weight, const void* bias, int64_t rows,
                               int64_t dim, float scale, float eps, int32_t type, int32_t state_type,
                               int32_t param_type, void* state_out, void* y, float* stats, void* codes, void* scales,
                               jn_stream_t stream) {
  return forward(state, x, weight, bias, rows, dim, scale, eps, type, state_type, param_type, state_out, y, stats,
                 true, codes, scales, stream);
}

size_t jn_layer_norm_backward_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows < 1 || dim < 1 || dim >= (1LL << 28)) return 0;
  return (size_t)part_count(rows, dim) * 2 * dim * sizeof(float);
}

int jn_layer_norm_backward(const void* state, const void* x, const void* weight, const float* stats,
                           const void* grad_state_out, const void* grad_y, int64_t rows, int64_t dim, float scale,
                           int32_t type, int32_t state_type, int32_t param_type, void* grad_state, void* grad_x,
                           void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                           jn_stream_t stream) {
  return backward(state, x, weight, stats, grad_state_out, grad_y, rows, dim, scale, type, state_type, param_type,
                  grad_state, grad_x, grad_weight, grad_bias, workspace, workspace_bytes, false, nullptr, nullptr,
                  stream);
}

int jn_layer_norm_backward_kept(const void* state, const void* codes, const void* scales, const void* weight,
                                const float* stats, const void* grad_state_out, const void* grad_y, int64_t rows,
                                int64_t dim, float scale, int32_t type, int32_t state_type, int32_t param_type,
                                void* grad_state, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                                size_t workspace_bytes, jn_stream_t stream) {
  return backward(state, nullptr, weight, stats, grad_state_out, grad_y, rows, dim, scale, type, state_type, param_type,
                  grad_state, grad_x, grad_weight, grad_bias, workspace, workspace_bytes, true, codes, scales, stream);
}

}  // extern "C"
