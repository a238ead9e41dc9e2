// Products with a microscaled operand (jn_mx_linear_*, jn_mx_weight_grad).
//
//   forward      y[m, n] = sum_k x[m, k] W[n, k] + b[n], W microscaled along k; x as it
//                is (mx_mixed_kernel), or microscaled along k too on its way in
//                (mx_linear_kernel, on the scaled matrix instructions)
//   gradients    c[m, n] = sum_r A(m, r) B[r, n] with B [r, n] microscaled along n
//                and A of ordinary numbers (mx_mixed_kernel): a frozen weight's input
//                gradient (A = grad_y [m, r], B = W) and a layer's weight gradient from
//                its kept input (A = grad_y^T, grad_y [r, m], B = x)
#include "../../include/jakal_net_hip.h"
#include "jn_internal.hpp"
#include "jn_mx.hpp"

namespace jakal {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));

// Tiles of a product's output over the workgroups: contiguous ranges per XCD,
// bands of 8 row tiles sweeping the columns.
struct TilePlace {
  int split, mi, ni;
  __device__ TilePlace(int tiles_m, int tiles_n) {
    const int id = xcd_swizzle(blockIdx.x, gridDim.x);
    const int per = tiles_m * tiles_n;
    split = id / per;
    const int t = id - split * per;
    constexpr int kBand = 8;
    const int band = t / (kBand * tiles_n);
    const int bm = min(kBand, tiles_m - band * kBand);
    const int tb = t - band * kBand * tiles_n;
    mi = band * kBand + tb % bm;
    ni = tb / bm;
  }
};

// ---- ordinary numbers by microscaled ones ---------------------------------------
// v_mfma_f32_16x16x32_bf16 over tiles of 64 x 64 to 256 x 256: microscaled values are
// bf16 values (at most four significant bits), and A is one, two or three bf16 terms
// that add up to it exactly (bf16, fp16, fp32), so every product is exact and the
// sums are fp32.  Both operands pass through registers on their way into LDS.  An
// operand whose rows run along r lies there as it does in memory ([row][r]); one
// whose rows run along m or n lies as [r][128] and is read transposed
// (ds_read_b64_tr_b16).
enum Product { kForward, kInputGrad, kWeightGrad, kPlainGrad };

struct MixedArgs {
  const void* a;          // [m][lda], or [r][lda] (weight gradient)
  const uint8_t* codes;   // B: [n][pitch] along r (forward), or [r][pitch] along n
  const uint8_t* scales;  // a byte a run, in the same order
  const void* bias;       // [n] or null (forward)
  void* out;              // [m][n] of the element type, or null: partial sums
  float* partial;         // [splits][m][ldp]
  void* bias_grad;        // [m]: sums of A over r (weight gradient), or null
  float* bias_partial;    // [splits][m]
  int64_t m, n, r;
  int64_t lda, ldp, pitch, runs;
  int64_t chunk;          // of r a split, a multiple of the slice
  int tiles_m, tiles_n;
};

constexpr int kPlain = -1;  // activations that are not microscaled

template <typename T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : std::is_same_v<T, f16_t> ? 2 : 1;
template <typename T>
constexpr int kSlice = kTerms<T> == 1 ? 64 : 32;

// The bf16 terms of two numbers, each pair in a word.
template <typename T>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[kTerms<T>]) {
  if constexpr (kTerms<T> == 3) {
    uint32_t h[2], m[2], l[2];
    const uint32_t u[2] = {__float_as_uint(a), __float_as_uint(b)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x3_split(u[i], h[i], m[i], l[i]);
      // an infinity or a NaN has no remainder, and a NaN must not lose its low bits
      if ((u[i] & 0x7F800000u) == 0x7F800000u) {
        m[i] = l[i] = 0;
        if (u[i] & 0x7FFFFFu) h[i] |= 0x400000u;
      }
    }
    w[0] = x3_pair(h[0], h[1]), w[1] = x3_pair(m[0], m[1]), w[2] = x3_pair(l[0], l[1]);
  } else {  // fp16: eight bits and the other three
    const uint32_t h0 = __float_as_uint(a) & 0xFFFF0000u, h1 = __float_as_uint(b) & 0xFFFF0000u;
    const bool f0 = fabsf(a) < __builtin_inff(), f1 = fabsf(b) < __builtin_inff();
    const uint32_t l0 = f0 ? __float_as_uint(a - __uint_as_float(h0)) : 0;
    const uint32_t l1 = f1 ? __float_as_uint(b - __uint_as_float(h1)) : 0;
    const uint32_t q0 = a != a ? 0x400000u : 0u, q1 = b != b ? 0x400000u : 0u;
    w[0] = x3_pair(h0 | q0, h1 | q1), w[1] = x3_pair(l0, l1);
  }
}

// A uniform stride that the compiler takes for new wherever it is asked for: it would keep
// the multiples of it that a loop needs in registers that the loop's operands need.
__device__ __forceinline__ uint32_t fresh(int64_t v) {
  uint32_t x = (uint32_t)v;
  asm volatile("" : "+s"(x));
  return x;
}

// Places in LDS, in bf16 elements, so that the lanes of one read fall on all banks.
// [row][SLICE] with the slice along the row: 16-byte chunks permuted by the row.
template <int SLICE>
__device__ __forceinline__ int lds_kc(int row, int chunk) {
  if constexpr (SLICE == 64) return row * 64 + ((chunk ^ (row >> 1)) & 7) * 8;
  else return row * 32 + ((chunk ^ -(row >> 2)) & 3) * 8;
}
// [r][WIDTH]: the 32-byte chunks of each 256 bytes permuted by the row.
template <int WIDTH>
__device__ __forceinline__ int lds_tr(int r, int chunk32) {
  return r * WIDTH + (chunk32 & ~7) * 16 + ((chunk32 ^ ((r & 3) | ((r >> 1) & 4))) & 7) * 16;
}

__device__ __forceinline__ shortx4 read_tr(const bf16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) shortx4*)(const_cast<bf16_t*>(p)));
}

// The bf16 kernel's [r][WIDTH]: rows of 32 bytes more, and 128 more every eight rows, so
// that four rows and those eight further on fall on different banks.  Sums of what a row
// and a column add, where a permutation would take an address for every tile.
constexpr int kPadEight = 64;
template <int WIDTH>
constexpr int kPadRow = WIDTH + 16;
template <int WIDTH>
constexpr int kPadPlane = 64 * kPadRow<WIDTH> + 8 * kPadEight;
template <int WIDTH>
__device__ __forceinline__ int lds_pad(int r, int c) {
  return r * kPadRow<WIDTH> + (r >> 3) * kPadEight + c;
}

// Eight consecutive r from r0 on of column c16 * 16 + (lane & 15), for lane group g: r0 = 8 g.
template <int WIDTH>
__device__ __forceinline__ bf16x8v fragment_tr(const bf16_t* plane, int r0, int c16, int lane) {
  const int i = lane & 15;
  const shortx4 a = read_tr(plane + lds_tr<WIDTH>(r0 + (i >> 2), c16) + (i & 3) * 4);
  const shortx4 b = read_tr(plane + lds_tr<WIDTH>(r0 + 4 + (i >> 2), c16) + (i & 3) * 4);
  typedef short shortx8 __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(bf16x8v, (shortx8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Four consecutive elements of an output row of n elements, from element c on.
template <typename T>
__device__ __forceinline__ void store_quad(T* p, int64_t c, int64_t n, const float (&v)[4]) {
  if (n % 4 == 0) {
    store_raw<T, 4>(p, v);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (c + q < n) p[q] = (T)v[q];
    }
  }
}
template <typename T>
__device__ __forceinline__ void load_bias(const T* bias, int64_t c, int64_t n, float (&b)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) b[q] = bias && c + q < n ? (float)bias[c + q] : 0.f;
}

// A wave's MT x NT tiles of outputs, the first at (m0, n0), plus the bias where there is
// one.  Rows of whole 16-byte packs go through the wave's part of LDS, GROUP tiles of rows
// by a line of 128 bytes (or all there is) at a time; others straight from the registers.
template <typename T, int NT>
constexpr int kLineTiles = NT * 16 * sizeof(T) > 128 ? 128 / (16 * (int)sizeof(T)) : NT;
template <typename T, int NT>
constexpr int kLineBytes = kLineTiles<T, NT> * 16 * (int)sizeof(T) + 16;  // sixteen more, so that rows begin on other banks

template <typename T, int MT, int NT, int GROUP>
__device__ __forceinline__ void store_tile(const floatx4 (&acc)[NT][MT], uint8_t* lds, const T* bias, T* out, int64_t m0,
                                           int64_t n0, int64_t rows, int64_t cols, int lane) {
  const int grp = lane >> 4, col = lane & 15;
  float b[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) load_bias(bias, n0 + i * 16 + grp * 4, cols, b[i]);
  if (cols * sizeof(T) % 16 != 0) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int64_t n = n0 + i * 16 + grp * 4;
      if (n >= cols) continue;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int64_t m = m0 + j * 16 + col;
        if (m >= rows) continue;
        const float v[4] = {acc[i][j][0] + b[i][0], acc[i][j][1] + b[i][1], acc[i][j][2] + b[i][2],
                            acc[i][j][3] + b[i][3]};
        store_quad(out + m * cols + n, n, cols, v);
      }
    }
    return;
  }
  constexpr int LT = kLineTiles<T, NT>, kRow = kLineBytes<T, NT>;
  constexpr int kChunks = LT * 16 * (int)sizeof(T) / 16, kLaneRows = kWave / kChunks;
  const int chunk = lane % kChunks, first = lane / kChunks;
#pragma unroll
  for (int j0 = 0; j0 < MT; j0 += GROUP) {
#pragma unroll
    for (int i0 = 0; i0 < NT; i0 += LT) {
#pragma unroll
      for (int j = j0; j < j0 + GROUP; ++j) {
#pragma unroll
        for (int i = i0; i < i0 + LT; ++i) {
          const float v[4] = {acc[i][j][0] + b[i][0], acc[i][j][1] + b[i][1], acc[i][j][2] + b[i][2],
                              acc[i][j][3] + b[i][3]};
          store_raw<T, 4>(reinterpret_cast<T*>(lds + ((j - j0) * 16 + col) * kRow) + (i - i0) * 16 + grp * 4, v);
        }
      }
      wave_lds_sync();
      const int64_t n = n0 + i0 * 16 + chunk * (16 / (int)sizeof(T));
#pragma unroll
      for (int r = 0; r < GROUP * 16; r += kLaneRows) {
        const int64_t m = m0 + j0 * 16 + r + first;
        const uint4 v = *reinterpret_cast<const uint4*>(lds + (r + first) * kRow + chunk * 16);
        if (m < rows && n < cols) *reinterpret_cast<uint4*>(out + m * cols + n) = v;
      }
      wave_lds_sync();
    }
  }
}

// Two elements of e4m3 or e2m1 as bf16, times the run's scale: one instruction.
template <int FORM, int WORD_HALF>
__device__ __forceinline__ uint32_t decode_pair(uint32_t code, float scale) {
  if constexpr (FORM == kE4m3)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code, scale, WORD_HALF));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, WORD_HALF));
}

// Eight elements of a row, `left` of them inside it (at most eight count): one access
// where they all are, whatever the row's alignment; zeros past the end.
template <typename T>
struct Eight {
  typedef T vec __attribute__((ext_vector_type(8)));
  typedef vec loose __attribute__((aligned(sizeof(T))));
  vec v;

  __device__ __forceinline__ void load(const T* p, int64_t left) {
    if (left >= 8) {
      v = *reinterpret_cast<const loose*>(p);
    } else {
      v = vec{};
#pragma unroll
      for (int i = 0; i < 7; ++i) {
        if (i < left) v[i] = p[i];
      }
    }
  }
};

// Loads straight into LDS, 16 or 4 bytes a lane, at `base` + lane * BYTES.  In assembly,
// since the compiler would wait for all of them before any later read of LDS: whoever
// reads waits itself (wait_loads, then the barrier).  They have no result registers.
typedef __attribute__((address_space(3))) const uint8_t lds_byte;
typedef int intx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t lds_offset(const uint8_t* p) { return (uint32_t)(uintptr_t)(lds_byte*)p; }

// The resource over [base, base + bytes), or its first 2^32 - 1 bytes: a tile's rows
// reach no further.  Empty where bytes is negative.
__device__ __forceinline__ intx4 rows_rsrc(const uint8_t* base, int64_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  return intx4{__builtin_amdgcn_readfirstlane((int)(uint32_t)p),
               __builtin_amdgcn_readfirstlane((int)((uint32_t)(p >> 32) & 0xFFFFu)),
               __builtin_amdgcn_readfirstlane((int)(uint32_t)max((int64_t)0, min(bytes, (int64_t)0xFFFFFFFF))), 0x00020000};
}

// `base` and the resource are uniform over the wave.
template <int BYTES>
__device__ __forceinline__ void load_lds(intx4 rs, uint32_t base, uint32_t offset) {
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(base), "v"(offset), "s"(rs)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(base), "v"(offset), "s"(rs)
                 : "memory", "m0");
}

// Until the wave's loads have landed and its reads of LDS are done.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// Tiles of TM x TN over WM x WN waves, LDS double buffered with the next slice in registers.
// For fp32, fp16 and rows that are no whole packs.  Splitting x into its terms and their way
// through LDS bound it: 1,531 x 383 x 4,099 fp32 forward 41 us (117 TFLOP/s; the library's
// fp32 product by dequantised weights 88 us), 128 x 2,048 x 16,384 fp32 53 us (the library
// 77).  fp16 is slower than the library's fp16 product by dequantised weights: 128 rows 40 us
// and 17, 1,024 rows 177 and 55.
template <typename T, Product P, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM* WN* kWave, 2) void mx_mixed_kernel(MixedArgs g) {
  constexpr int FORM = P == kWeightGrad ? kE4m3 : kE2m1;
  constexpr bool A_R = P != kWeightGrad, B_R = P == kForward;  // rows along r
  constexpr int TERMS = kTerms<T>, SLICE = kSlice<T>, THREADS = WM * WN * kWave;
  constexpr int kA = TM * SLICE, kB = TN * SLICE;  // elements of a plane
  constexpr int kStage = TERMS * kA + kB;
  constexpr int UA = kA / 8 / THREADS, UB = kB / 8 / THREADS;  // units of eight elements a thread
  constexpr int MT = TM / WM / 16, NT = TN / WN / 16;
  __shared__ __align__(16) bf16_t smem[2 * kStage];

  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
  const int grp = lane >> 4, col = lane & 15;
  const int wm = wave / WN, wn = wave % WN;
  const TilePlace at(g.tiles_m, g.tiles_n);
  const int64_t m0 = (int64_t)at.mi * TM, n0 = (int64_t)at.ni * TN;
  const int64_t rbeg = at.split * g.chunk, rend = min(g.r, rbeg + g.chunk);
  const T* abase = static_cast<const T*>(g.a);
  const bool sums = P == kWeightGrad && g.bias_partial && at.ni == 0;

  // one slice in registers
  Eight<T> ra[UA];
  uint2 rb[UB];
  int rs[UB];
  auto load = [&](int64_t r0) {
#pragma unroll
    for (int u = 0; u < UA; ++u) {
      const int id = tid + THREADS * u;
      const int64_t row = A_R ? m0 + id / (SLICE / 8) : r0 + id / (TM / 8);
      const int64_t c = A_R ? r0 + id % (SLICE / 8) * 8 : m0 + id % (TM / 8) * 8;
      ra[u].load(abase + row * g.lda + c, row < (A_R ? g.m : rend) ? (A_R ? rend : g.m) - c : 0);
    }
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const int id = tid + THREADS * u;
      const int64_t row = B_R ? n0 + id / (SLICE / 8) : r0 + id / (TN / 8);
      const int64_t e = B_R ? r0 + id % (SLICE / 8) * 8 : n0 + id % (TN / 8) * 8;
      rb[u] = uint2{0, 0}, rs[u] = 127;
      if (row < (B_R ? g.n : rend) && e < g.runs * kMxRun) {
        if constexpr (FORM == kE4m3) rb[u] = *reinterpret_cast<const uint2*>(g.codes + row * g.pitch + e);
        else rb[u].x = *reinterpret_cast<const uint32_t*>(g.codes + row * g.pitch + e / 2);
        rs[u] = g.scales[row * g.runs + e / kMxRun];
      }
    }
  };
  float total[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto store = [&](bf16_t* stage) {
#pragma unroll
    for (int u = 0; u < UA; ++u) {
      const int id = tid + THREADS * u;
      bf16_t* p = stage + (A_R ? lds_kc<SLICE>(id / (SLICE / 8), id % (SLICE / 8))
                               : lds_tr<TM>(id / (TM / 8), id % (TM / 8) / 2) + id % 2 * 8);
      if (sums) {
#pragma unroll
        for (int j = 0; j < 8; ++j) total[j] += (float)ra[u].v[j];
      }
      if constexpr (TERMS == 1) {
        *reinterpret_cast<typename Eight<T>::vec*>(p) = ra[u].v;
      } else {
        uint32_t w[4][TERMS];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_pair<T>((float)ra[u].v[2 * j], (float)ra[u].v[2 * j + 1], w[j]);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
          *reinterpret_cast<uint4*>(p + t * kA) = make_uint4(w[0][t], w[1][t], w[2][t], w[3][t]);
      }
    }
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const int id = tid + THREADS * u;
      const float scale = mx_scale(rs[u]);
      uint4 d;
      if constexpr (FORM == kE4m3)
        d = make_uint4(decode_pair<FORM, 0>(rb[u].x, scale), decode_pair<FORM, 1>(rb[u].x, scale),
                       decode_pair<FORM, 0>(rb[u].y, scale), decode_pair<FORM, 1>(rb[u].y, scale));
      else
        d = make_uint4(decode_pair<FORM, 0>(rb[u].x, scale), decode_pair<FORM, 1>(rb[u].x, scale),
                       decode_pair<FORM, 2>(rb[u].x, scale), decode_pair<FORM, 3>(rb[u].x, scale));
      *reinterpret_cast<uint4*>(stage + TERMS * kA +
                                (B_R ? lds_kc<SLICE>(id / (SLICE / 8), id % (SLICE / 8))
                                     : lds_tr<TN>(id / (TN / 8), id % (TN / 8) / 2) + id % 2 * 8)) = d;
    }
  };

  floatx4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int slices = rend > rbeg ? (int)((rend - rbeg + SLICE - 1) / SLICE) : 0;
  if (slices > 0) {
    load(rbeg);
    store(smem);
  }
  __syncthreads();
  for (int s = 0; s < slices; ++s) {
    const bf16_t* stage = smem + (s & 1) * kStage;
    if (s + 1 < slices) load(rbeg + (int64_t)(s + 1) * SLICE);
#pragma unroll
    for (int k = 0; k < SLICE / 32; ++k) {
      bf16x8v b[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if constexpr (B_R)
          b[i] = *reinterpret_cast<const bf16x8v*>(stage + TERMS * kA +
                                                   lds_kc<SLICE>(wn * (TN / WN) + i * 16 + col, k * 4 + grp));
        else
          b[i] = fragment_tr<TN>(stage + TERMS * kA, k * 32 + grp * 8, wn * NT + i, lane);
      }
#pragma unroll
      for (int t = TERMS - 1; t >= 0; --t) {  // the smallest terms first
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          bf16x8v a;
          if constexpr (A_R)
            a = *reinterpret_cast<const bf16x8v*>(stage + t * kA +
                                                  lds_kc<SLICE>(wm * (TM / WM) + j * 16 + col, k * 4 + grp));
          else
            a = fragment_tr<TM>(stage + t * kA, k * 32 + grp * 8, wm * MT + j, lane);
#pragma unroll
          for (int i = 0; i < NT; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[i], a, acc[i][j], 0, 0, 0);
        }
      }
    }
    if (s + 1 < slices) store(smem + ((s + 1) & 1) * kStage);
    __syncthreads();
  }

  // a lane holds four consecutive n of one m in each tile
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int64_t n = n0 + wn * (TN / WN) + i * 16 + grp * 4;
    if (n >= g.n) continue;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (P == kForward && g.out) load_bias(static_cast<const T*>(g.bias), n, g.n, bias);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int64_t m = m0 + wm * (TM / WM) + j * 16 + col;
      if (m >= g.m) continue;
      if (g.out) {
        const float v[4] = {acc[i][j][0] + bias[0], acc[i][j][1] + bias[1], acc[i][j][2] + bias[2],
                            acc[i][j][3] + bias[3]};
        store_quad(static_cast<T*>(g.out) + m * g.n + n, n, g.n, v);
      } else {
        *reinterpret_cast<floatx4*>(g.partial + ((int64_t)at.split * g.m + m) * g.ldp + n) = acc[i][j];
      }
    }
  }
  if (sums) {  // the threads that had the same eight columns, in order
    float* lds = reinterpret_cast<float*>(smem);
    constexpr int kSame = THREADS / (TM / 8);
    static_assert(UA == 0 || THREADS % (TM / 8) == 0, "a thread keeps its columns");
#pragma unroll
    for (int j = 0; j < 8; ++j) lds[(tid / (TM / 8)) * TM + tid % (TM / 8) * 8 + j] = total[j];
    __syncthreads();
    if (tid < TM && m0 + tid < g.m) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < kSame; ++i) t += lds[i * TM + tid];
      g.bias_partial[(int64_t)at.split * g.m + m0 + tid] = t;
    }
  }
}

// The same for bf16 A with rows of whole, aligned 16-byte packs: tiles of TM x TN over
// WM x WN waves.  A slice is two half steps of 32 r.  Its operands are read from LDS while
// the half step before is multiplied, each as soon as its register is free; the slice
// after lies in registers by then and goes to the other stage meanwhile, and AHEAD slices
// after that are on their way from memory.  B may be plain bf16 too (kPlainGrad: a linear
// layer's input gradient).
// The widest tiles keep the matrix units at 1,220 TFLOP/s over long sums (8,192 x 2,048 over
// 8,192 225 us, the library by dequantised weights 202); what is left is a tile's start and
// its outputs' way out, with no other workgroup on the CU (8,192 x 2,048 x 16,384 forward 490
// us, 1,110 TFLOP/s, the library 404).  A quarter less LDS traffic (B there as its codes) and
// the barrier under the first row of products gained 2 %.  The narrow ones wait for each other once a slice:
// 0.53 to 0.85 us whatever they multiply, and loads further ahead (four slices) or twice the
// waves changed nothing.  256 x 256 takes all 256 registers: the forward keeps one more in
// scratch and the input gradient two.
template <Product P, int TM, int TN, int WM, int WN, int AHEAD>
__global__ __launch_bounds__(WM* WN* kWave, 2) void mx_bf16_kernel(MixedArgs g) {
  constexpr int FORM = P == kWeightGrad ? kE4m3 : kE2m1;
  constexpr bool A_R = P != kWeightGrad, B_R = P == kForward, B_PLAIN = P == kPlainGrad;
  // sums of A over r, where there are registers for them
  constexpr bool SUMS = P == kWeightGrad && TM < 256;
  constexpr int SLICE = 64, THREADS = WM * WN * kWave;
  constexpr int UA = TM * SLICE / 8 / THREADS, UB = TN * SLICE / 8 / THREADS;  // units of eight elements a thread
  constexpr int kA = A_R ? TM * SLICE : kPadPlane<TM>, kB = B_R ? TN * SLICE : kPadPlane<TN>, kStage = kA + kB;
  constexpr int MT = TM / WM / 16, NT = TN / WN / 16;
  __shared__ __align__(16) bf16_t smem[2 * kStage];

  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
  const int grp = lane >> 4, col = lane & 15;
  const int wm = wave / WN, wn = wave % WN;
  const TilePlace at(g.tiles_m, g.tiles_n);
  const int64_t m0 = (int64_t)at.mi * TM, n0 = (int64_t)at.ni * TN;
  const int64_t rbeg = at.split * g.chunk, rend = min(g.r, rbeg + g.chunk);
  const int slices = rend > rbeg ? (int)((rend - rbeg + SLICE - 1) / SLICE) : 0;

  // A thread's units of a slice are `kStep` rows apart: rows of m or n (ROWS_R) or of r.
  // What lies past the last row, or past r's end, is out of range and reads as zeros; m
  // and n past the end within rows of r are the next row's numbers (their outputs are
  // not written).
  constexpr int UR = SLICE / 8, UTA = TM / 8, UTB = TN / 8;  // units of a row along r, and across
  const int urow = tid / UR, uunit = tid % UR;
  const int arow = tid / UTA, aunit = tid % UTA, brow = tid / UTB, bunit = tid % UTB;
  constexpr int kStepR = THREADS / UR, kStepA = THREADS / UTA, kStepB = THREADS / UTB;
  struct Slice {
    uint4 a[UA];
    u32x4_nt b[UB];
    uint32_t s[UB];
  } held[AHEAD];
  // `first`: the operand's first row and first unit here, `bytes` a row's, `unit` a unit's
  const auto place = [&](bool rows_r, const void* base, int64_t rows, int64_t first, int64_t c, int64_t bytes, int left) {
    const int64_t skip = first * bytes + c;
    const int64_t end = rows_r ? rows * bytes : min(rows, first + left) * bytes;
    return make_rsrc(static_cast<const char*>(base) + skip, (uint32_t)max((int64_t)0, min(end - skip, (int64_t)0x7FFFFFFF)));
  };
  auto load = [&](int s, Slice& to) {
    const int64_t r0 = rbeg + (int64_t)s * SLICE;
    const int left = (int)max((int64_t)0, min((int64_t)SLICE, rend - r0));  // of r in the slice
    const uint32_t skip = uunit * 8 < left ? 0u : kOobOffset;               // of a unit along r
    const auto rsa = A_R ? place(true, g.a, g.m, m0, r0 * 2, g.lda * 2, left) : place(false, g.a, g.r, r0, m0 * 2, g.lda * 2, left);
    const uint32_t lda = fresh(g.lda * 2);
    const uint32_t oa = A_R ? (uint32_t)urow * lda + uunit * 16 + skip : (uint32_t)arow * lda + aunit * 16;
#pragma unroll
    for (int u = 0; u < UA; ++u)
      to.a[u] = __builtin_bit_cast(
          uint4, __builtin_amdgcn_raw_buffer_load_b128(rsa, oa + u * (A_R ? kStepR : kStepA) * lda, 0, 0));
    if constexpr (B_PLAIN) {
      const uint32_t ldb = fresh(g.n * 2), ob = (uint32_t)brow * ldb + bunit * 16;
      const auto rsb = place(false, g.codes, g.r, r0, n0 * 2, g.n * 2, left);
#pragma unroll
      for (int u = 0; u < UB; ++u) to.b[u] = __builtin_amdgcn_raw_buffer_load_b128(rsb, ob + u * kStepB * ldb, 0, 0);
    } else {
      constexpr int UNIT = FORM == kE4m3 ? 8 : 4;  // bytes of a unit's codes
      const uint32_t pitch = fresh(g.pitch), runs = fresh(g.runs);
      const auto rsb = B_R ? place(true, g.codes, g.n, n0, r0 / 8 * UNIT, g.pitch, left)
                           : place(false, g.codes, g.r, r0, n0 / 8 * UNIT, g.pitch, left);
      const auto rss = B_R ? place(true, g.scales, g.n, n0, r0 / kMxRun, g.runs, left)
                           : place(false, g.scales, g.r, r0, n0 / kMxRun, g.runs, left);
      const uint32_t ob = B_R ? (uint32_t)urow * pitch + uunit * UNIT + skip : (uint32_t)brow * pitch + bunit * UNIT;
      const uint32_t os = B_R ? (uint32_t)urow * runs + uunit / 4 + skip : (uint32_t)brow * runs + bunit / 4;
#pragma unroll
      for (int u = 0; u < UB; ++u) {
        const uint32_t step = u * (B_R ? kStepR : kStepB);
        if constexpr (FORM == kE4m3) {
          const auto v = __builtin_amdgcn_raw_buffer_load_b64(rsb, ob + step * pitch, 0, 0);
          to.b[u][0] = v[0], to.b[u][1] = v[1];
        } else {
          to.b[u][0] = __builtin_amdgcn_raw_buffer_load_b32(rsb, ob + step * pitch, 0, 0);
        }
        to.s[u] = __builtin_amdgcn_raw_buffer_load_b8(rss, os + step * runs, 0, 0);
      }
    }
  };
  // (a unit's row is a whole number of eight rows and of the chunks' permutation further on)
  const int along = lds_kc<SLICE>(urow, uunit);
  const int aplace = A_R ? along : lds_pad<TM>(arow, aunit * 8), bplace = B_R ? along : lds_pad<TN>(brow, bunit * 8);
  constexpr int kNextA = A_R ? kStepR * SLICE : kStepA * kPadRow<TM> + kStepA / 8 * kPadEight;
  constexpr int kNextB = B_R ? kStepR * SLICE : kStepB * kPadRow<TN> + kStepB / 8 * kPadEight;
  static_assert(kStepR % 16 == 0 && kStepA % 8 == 0 && kStepB % 8 == 0, "a unit's place is the first one's and a constant");
  float total[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto store_a = [&](int stage, int u, const Slice& from) {
    *reinterpret_cast<uint4*>(smem + stage + aplace + u * kNextA) = from.a[u];
    if constexpr (SUMS) {
      const auto v = __builtin_bit_cast(bf16x8v, from.a[u]);
#pragma unroll
      for (int j = 0; j < 8; ++j) total[j] += (float)v[j];
    }
  };
  auto store_b = [&](int stage, int u, const Slice& from) {
    const u32x4_nt b = from.b[u];
    uint4 d;
    if constexpr (B_PLAIN) {
      d = make_uint4(b[0], b[1], b[2], b[3]);
    } else {
      const float scale = mx_scale((int)from.s[u]);
      if constexpr (FORM == kE4m3)
        d = make_uint4(decode_pair<FORM, 0>(b[0], scale), decode_pair<FORM, 1>(b[0], scale),
                       decode_pair<FORM, 0>(b[1], scale), decode_pair<FORM, 1>(b[1], scale));
      else
        d = make_uint4(decode_pair<FORM, 0>(b[0], scale), decode_pair<FORM, 1>(b[0], scale),
                       decode_pair<FORM, 2>(b[0], scale), decode_pair<FORM, 3>(b[0], scale));
    }
    *reinterpret_cast<uint4*>(smem + stage + kA + bplace + u * kNextB) = d;
  };

  bf16x8v a[MT], b[NT];  // one half step's operands
  // one address an operand and constants: sixteen rows further on the chunks are permuted
  // alike, and the other half step's are four chunks further on
  const auto read = [&](bool rows_r, int row, int origin, int base, int k, int t) -> bf16x8v {
    if (rows_r) return *reinterpret_cast<const bf16x8v*>(smem + origin + (base ^ (32 * k)) + t * 16 * SLICE);
    const bf16_t* p = smem + origin + base + k * (32 * row + 4 * kPadEight) + t * 16;
    const shortx4 lo = read_tr(p), hi = read_tr(p + 4 * row);
    typedef short shortx8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(bf16x8v, (shortx8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  const int am = wm * (TM / WM), bn = wn * (TN / WN);  // the wave's part of the tile
  const int abase = A_R ? lds_kc<SLICE>(am + col, grp) : lds_pad<TM>(grp * 8 + (col >> 2), am + (col & 3) * 4);
  const int bbase = B_R ? lds_kc<SLICE>(bn + col, grp) : lds_pad<TN>(grp * 8 + (col >> 2), bn + (col & 3) * 4);
  auto read_a = [&](int stage, int k, int j) { a[j] = read(A_R, kPadRow<TM>, stage, abase, k, j); };
  auto read_b = [&](int stage, int k, int i) { b[i] = read(B_R, kPadRow<TN>, stage + kA, bbase, k, i); };
  floatx4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto half = [&](int next, int k, auto then) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[i], a[j], acc[i][j], 0, 0, 0);
        if (i == NT - 1) read_a(next, k, j);
      }
      then(i);
      read_b(next, k, i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Slice s, whose first operands are in registers; the slice after it, on hand in `after`.
  auto step = [&](int s, int cur, int next, Slice& after) {
    half(cur, 1, [&](int i) {
#pragma unroll
      for (int u = i * UA / NT; u < (i + 1) * UA / NT; ++u) store_a(next, u, after);
#pragma unroll
      for (int u = i * UB / NT; u < (i + 1) * UB / NT; ++u) store_b(next, u, after);
    });
    load(s + 1 + AHEAD, after);  // (nothing past the last)
    // every wave has this slice's operands in registers, and has stored its part of the next
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    half(next, 0, [](int) {});
  };
  if (slices > 0) {
    load(0, held[0]);
#pragma unroll
    for (int u = 0; u < UA; ++u) store_a(0, u, held[0]);
#pragma unroll
    for (int u = 0; u < UB; ++u) store_b(0, u, held[0]);
#pragma unroll
    for (int i = 1; i <= AHEAD; ++i) load(i, held[i % AHEAD]);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MT; ++j) read_a(0, 0, j);
#pragma unroll
    for (int i = 0; i < NT; ++i) read_b(0, 0, i);
  }
  if constexpr (AHEAD == 1) {
    for (int s = 0; s < slices; ++s) step(s, (s & 1) * kStage, kStage - (s & 1) * kStage, held[0]);
  } else {
    static_assert(AHEAD % 2 == 0, "a slice's stage is its number's parity");
    for (int s = 0; s < slices; s += AHEAD) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (s + i < slices) step(s + i, (i & 1) * kStage, kStage - (i & 1) * kStage, held[(i + 1) % AHEAD]);
      }
    }
  }

  constexpr int kWaveBytes = 2 * kStage * (int)sizeof(bf16_t) / (WM * WN);
  constexpr int GROUP = MT < 4 ? MT : 4;
  static_assert(GROUP * 16 * kLineBytes<float, NT> <= kWaveBytes && GROUP * 16 * kLineBytes<bf16_t, NT> <= kWaveBytes,
                "a wave's part of LDS");
  uint8_t* const lds = reinterpret_cast<uint8_t*>(smem) + wave * kWaveBytes;
  __syncthreads();  // LDS is used anew
  if (g.out)
    store_tile<bf16_t, MT, NT, GROUP>(acc, lds, P == kForward ? static_cast<const bf16_t*>(g.bias) : nullptr,
                                  static_cast<bf16_t*>(g.out), m0 + am, n0 + bn, g.m, g.n, lane);
  else
    store_tile<float, MT, NT, GROUP>(acc, lds, nullptr, g.partial + (int64_t)at.split * g.m * g.ldp, m0 + am, n0 + bn,
                                 g.m, g.ldp, lane);
  if constexpr (SUMS) {  // the threads that had the same eight columns, in order
    if (!g.bias_partial || at.ni != 0) return;
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[arow * TM + aunit * 8 + j] = total[j];
    __syncthreads();
    if (tid < TM && m0 + tid < g.m) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < kStepA; ++i) t += sums[i * TM + tid];
      g.bias_partial[(int64_t)at.split * g.m + m0 + tid] = t;
    }
  }
}

// The forward of bf16 x whose rows are whole steps of 128 k, where there are few: tiles of
// TM x TN over 2 x 2 waves, a column of them half the outputs, a row of them half of each
// run of 32 k (their sums join at the end).  x, W's codes and scales go straight into LDS,
// STAGES - 1 steps ahead, and W's are decoded as they are read, so that neither a register
// nor a wait lies between memory and LDS, and two workgroups fit a CU.  The four bf16
// operands of a step take k as a run has them: lane group g eight k of run g each.  What
// bounds it are those loads: one workgroup a CU moves 35 KB a us, with one step or three on
// their way, two 52 (so two small ones, not one with more stages: 128 x 2,048 x 16,384 with
// four stages 24 us, with two 20).
template <int TM, int TN, int STAGES>
__global__ __launch_bounds__(256, 2) void mx_direct_kernel(MixedArgs g) {
  constexpr int STEP = 128, MT = TM / 16, NT = TN / 32;
  constexpr int XU = TM / 16, WU = TN / 64;  // 16-byte loads a lane and step, four and sixteen rows each
  constexpr int kX = TM * STEP * 2, kW = TN * STEP / 2, kS = TN * 4, kStage = kX + kW + kS;
  constexpr int kLoads = XU + WU + 1;
  __shared__ __align__(16) uint8_t smem[STAGES * kStage];

  const int lane = lane_id(), wave = wave_id();
  const int grp = lane >> 4, col = lane & 15;
  const int wn = wave & 1, half = wave >> 1;
  const TilePlace at(g.tiles_m, g.tiles_n);
  const int64_t m0 = (int64_t)at.mi * TM, n0 = (int64_t)at.ni * TN;
  const int mrows = (int)min((int64_t)TM, g.m - m0), nrows = (int)min((int64_t)TN, g.n - n0);
  const int64_t rbeg = at.split * g.chunk, rend = min(g.r, rbeg + g.chunk);
  const int steps = (int)((rend - rbeg) / STEP);

  // A row's sixteen chunks of 16 bytes permuted so that lanes that are read together
  // (rows 0-3 and 12-15 of one group, 4-11 of the next) fall on all banks.
  const auto turn = [](int row) { return (row & 11) | (row >> 1 & 4); };
  const int xrow = wave * 4 + lane / 16, xchunk = (lane % 16) ^ turn(xrow & 15);
  uint32_t ox[XU];
#pragma unroll
  for (int u = 0; u < XU; ++u) ox[u] = (uint32_t)min(u * 16 + xrow, mrows - 1) * (uint32_t)(g.lda * 2) + xchunk * 16;
  uint32_t ow[WU];
#pragma unroll
  for (int u = 0; u < WU; ++u)
    ow[u] = (uint32_t)min(u * 64 + wave * 16 + lane / 4, nrows - 1) * (uint32_t)g.pitch + lane % 4 * 16;
  const int srows = wave % WU * 64;
  const uint32_t os = (uint32_t)min(srows + lane, nrows - 1) * (uint32_t)g.runs;
  const uint32_t lds = lds_offset(smem);
  auto load = [&](int step, uint32_t stage) {
    const int64_t k = rbeg + (int64_t)step * STEP;
    const bool any = step < steps;  // (nothing past the last)
    const auto rows = [&](const uint8_t* base, int64_t skip, int64_t end) {
      return rows_rsrc(base + skip, any ? end - skip : 0);
    };
    const auto rx = rows(static_cast<const uint8_t*>(g.a), m0 * g.lda * 2 + k * 2, g.m * g.lda * 2);
    const auto rw = rows(g.codes, n0 * g.pitch + k / 2, g.n * g.pitch);
    const auto rs = rows(g.scales, n0 * g.runs + k / kMxRun, g.n * g.runs);
#pragma unroll
    for (int u = 0; u < XU; ++u) load_lds<16>(rx, lds + stage + (u * 4 + wave) * 1024, ox[u]);
#pragma unroll
    for (int u = 0; u < WU; ++u) load_lds<16>(rw, lds + stage + kX + (u * 4 + wave) * 1024, ow[u]);
    load_lds<4>(rs, lds + stage + kX + kW + srows * 4, os);  // (every wave, so that each has as many loads)
  };

  floatx4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int wat = kX + (wn * (TN / 2) + col) * 64 + grp * 16 + half * 8;
  const int sat = kX + kW + (wn * (TN / 2) + col) * 4 + grp;
  const int xat[2] = {col * 256 + ((grp * 4 + half * 2) ^ turn(col)) * 16, col * 256 + ((grp * 4 + half * 2 + 1) ^ turn(col)) * 16};

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(i, i * kStage);
  uint32_t cur = 0, behind = (STAGES - 1) * kStage;  // the stage of this step, and of the one before
  for (int s = 0; s < steps; ++s) {
    // this step's loads have landed and the reads of the one before are done, for all waves
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads * (STAGES - 2)) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    load(s + STAGES - 1, behind);
    const uint8_t* const stage = smem + cur;
    uint2 w[NT];
    float scale[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      w[i] = *reinterpret_cast<const uint2*>(stage + wat + i * 16 * 64);
      scale[i] = mx_scale(stage[sat + i * 16 * 4]);
    }
    bf16x8v x[2][MT];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int j = 0; j < MT; ++j) x[q][j] = *reinterpret_cast<const bf16x8v*>(stage + xat[q] + j * 16 * 256);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      bf16x8v b[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint32_t code = q ? w[i].y : w[i].x;
        b[i] = __builtin_bit_cast(bf16x8v, make_uint4(decode_pair<kE2m1, 0>(code, scale[i]), decode_pair<kE2m1, 1>(code, scale[i]),
                                                      decode_pair<kE2m1, 2>(code, scale[i]), decode_pair<kE2m1, 3>(code, scale[i])));
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[i], x[q][j], acc[i][j], 0, 0, 0);
      }
    }
    behind = cur;
    cur = cur == (STAGES - 1) * kStage ? 0 : cur + kStage;
  }

  constexpr int kWaveBytes = NT * MT * kWave * 16, GROUP = 2;
  static_assert(2 * kWaveBytes <= STAGES * kStage && GROUP * 16 * kLineBytes<float, NT> <= kWaveBytes, "LDS to join in");
  wait_loads();     // those past the last step too:
  __syncthreads();  // LDS is used anew
  uint8_t* const mine = smem + wn * kWaveBytes;
  if (half == 1) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) *reinterpret_cast<floatx4*>(mine + ((i * MT + j) * kWave + lane) * 16) = acc[i][j];
  }
  __syncthreads();
  if (half == 1) return;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] += *reinterpret_cast<const floatx4*>(mine + ((i * MT + j) * kWave + lane) * 16);
  wave_lds_sync();
  if (g.out)
    store_tile<bf16_t, MT, NT, GROUP>(acc, mine, static_cast<const bf16_t*>(g.bias), static_cast<bf16_t*>(g.out), m0,
                                      n0 + wn * (TN / 2), g.m, g.n, lane);
  else
    store_tile<float, MT, NT, GROUP>(acc, mine, nullptr, g.partial + (int64_t)at.split * g.m * g.ldp, m0, n0 + wn * (TN / 2),
                                     g.m, g.ldp, lane);
}

// The splits' sums in order, rounded once.  One thread four elements of a row.
template <typename T>
__global__ __launch_bounds__(256) void mx_sum_kernel(MixedArgs g, int splits) {
  const int64_t quads = g.ldp / 4, total = g.partial ? g.m * quads : 0;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id < total) {
    const int64_t m = id / quads, n = (id - m * quads) * 4;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s)
      v += *reinterpret_cast<const floatx4*>(g.partial + ((int64_t)s * g.m + m) * g.ldp + n);
    float w[4];
    load_bias(static_cast<const T*>(g.bias), n, g.n, w);
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] += v[q];
    store_quad(static_cast<T*>(g.out) + m * g.n + n, n, g.n, w);
  } else if (g.bias_partial && id - total < g.m) {
    const int64_t m = id - total;
    float t = 0.f;
    for (int s = 0; s < splits; ++s) t += g.bias_partial[(int64_t)s * g.m + m];
    static_cast<T*>(g.bias_grad)[m] = (T)t;
  }
}

// ---- sums over rows -------------------------------------------------------------
// A thread sums one column, or a 16-byte pack of them, over a slab of rows, a second
// launch the slabs in order.
constexpr int64_t kSlabRows = 32, kSlabs = 256;

int64_t sum_slabs(int64_t rows) { return std::min(kSlabs, (rows + kSlabRows - 1) / kSlabRows); }

template <typename T, int W>
__global__ __launch_bounds__(256) void column_sums_kernel(const T* x, int64_t rows, int64_t dim, int64_t each,
                                                          float* partial) {
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * W;
  if (c >= dim) return;
  const int64_t beg = blockIdx.y * each, end = min(rows, beg + each);
  float t[W] = {};
#pragma unroll 8
  for (int64_t r = beg; r < end; ++r) {
    Raw<T, W> raw;
    raw.load(x + r * dim + c);
    float v[W];
    raw.unpack(v);
#pragma unroll
    for (int i = 0; i < W; ++i) t[i] += v[i];
  }
#pragma unroll
  for (int i = 0; i < W; ++i) partial[blockIdx.y * dim + c + i] = t[i];
}

// 64 columns a workgroup, its waves a quarter of the slabs each (256 slabs by one thread a
// column took 60 us).
template <typename T>
__global__ __launch_bounds__(256) void columns_join_kernel(const float* partial, int64_t dim, int slabs, T* sums) {
  __shared__ float lds[4][kWave];
  const int64_t c = (int64_t)blockIdx.x * kWave + lane_id();
  float t = 0.f;
  if (c < dim) {
#pragma unroll 16
    for (int s = wave_id(); s < slabs; s += 4) t += partial[s * dim + c];
  }
  lds[wave_id()][lane_id()] = t;
  __syncthreads();
  if (wave_id() == 0 && c < dim) sums[c] = (T)(((lds[0][lane_id()] + lds[1][lane_id()]) + lds[2][lane_id()]) + lds[3][lane_id()]);
}

template <typename T>
int launch_column_sums(const void* x, int64_t rows, int64_t dim, float* partial, void* sums, hipStream_t s) {
  const int64_t slabs = sum_slabs(rows), each = (rows + slabs - 1) / slabs;
  JN_PROFILE("column_sums_kernel", s);
  constexpr int W = 16 / sizeof(T);
  const T* const p = static_cast<const T*>(x);
  if (dim % W == 0 && aligned16(x))
    hipLaunchKernelGGL((column_sums_kernel<T, W>), dim3((unsigned)((dim / W + 255) / 256), (unsigned)slabs), dim3(256), 0,
                       s, p, rows, dim, each, partial);
  else
    hipLaunchKernelGGL((column_sums_kernel<T, 1>), dim3((unsigned)((dim + 255) / 256), (unsigned)slabs), dim3(256), 0, s,
                       p, rows, dim, each, partial);
  JN_LAUNCH_CHECK();
  hipLaunchKernelGGL(columns_join_kernel<T>, dim3((unsigned)((dim + kWave - 1) / kWave)), dim3(256), 0, s, partial, dim,
                     (int)slabs, static_cast<T*>(sums));
  JN_LAUNCH_CHECK();
  return kOk;
}

// Tiles of a product's output and splits of its sum by what they were measured to cost (in
// us): a slice's time by how many workgroups a CU has, and for more than one split a second
// launch and the partial sums' way to memory and back.  A launch, a tile's start and its
// outputs' way out are not in it, so that it is near over long sums (input gradient of 1,024
// x 2,048 over 16,384 77.6 for 76 us, weight gradient of 8,192 x 512 x 2,048 35.8 for 38.4)
// and short over few slices and many outputs (forward of 1,024 x 512 x 2,048 4.0 for 8.6, of
// 1,024 x 2,048 x 16,384 51 for 63, of 8,192 rows 410 for 486; the head's weight gradient 51
// for 74), where the tiles' order by it is not always the measured one (192 x 2,048 x 16,384
// takes 27 us in tiles of 64 x 64, 256 rows 24 in tiles of 128 x 64).
struct TileCost {
  int m, n;
  double least, first, each;  // of a slice: max(least, first + each * workgroups a CU)
  int slice = 64;             // of r, for bf16
  bool direct = false;        // mx_direct_kernel
};
// bf16 rows of whole packs (mx_bf16_kernel).  Wide tiles feed the matrix units, narrow ones
// keep more CUs busy and cost less each: 128 x 2,048 x 16,384 forward with tiles of 256 x
// 256, 128 x 128, 128 x 64 and 64 x 64 55, 29, 23 and 23 us, 512 x 2,048 x 16,384 56, 44, 56
// and 65 us; the weight gradient of 1,024 x 512 x 2,048 32, 22, 18 and 14 us.
constexpr TileCost kPackedTiles[] = {
    {256, 256, 0, 0, 1.6}, {128, 128, 0.85, 0.41, 0.44}, {128, 64, 0.62, 0.1, 0.385}, {64, 64, 0.53, 0.13, 0.235}};
// Forward rows of whole steps of 128 (mx_direct_kernel; the others' least beside it): 128 x
// 2,048 x 16,384 19 and 23 us, 256 x 2,048 x 16,384 26 and 31, 1,024 x 2,048 x 2,048 18 and
// 23, 512 x 2,048 x 16,384 48 and 44.
constexpr TileCost kDirectTiles[] = {{128, 64, 1.0, 0.1, 0.67, 128, true}, {64, 64, 0.62, 0.15, 0.43, 128, true}};
// others (mx_mixed_kernel)
constexpr TileCost mixed_tile(int32_t type) {
  return type == kTypeF32 ? TileCost{128, 128, 1.3, 0.4, 0.9}
                          : TileCost{128, 128, 1.3, 0.7, type == kTypeF16 ? 0.6 : 0.4};
}

// Which tiles, and how many splits of the sum.
struct MixedPlan {
  TileCost tile;
  bool packed;  // mx_bf16_kernel's
  int tiles_m, tiles_n, splits;
  int64_t chunk, ldp;
  size_t partial_bytes, bias_bytes;

  bool wide() const { return tile.m == 256; }

  MixedPlan(Product p, int64_t m, int64_t n, int64_t r, int32_t type, bool bias) {
    // A's rows of whole packs of 16 bytes, and offsets of a tile's rows below 2^31
    const int64_t lda = p == kWeightGrad ? m : r;
    packed = type == kTypeBf16 && lda % 8 == 0 && lda < (1 << 21) && n < (1 << 21) && (p != kPlainGrad || n % 8 == 0);
    double least = 1e300;
    const auto consider = [&](const TileCost& c) {
      const int slice = type == kTypeBf16 ? c.slice : kSlice<float>;
      const int64_t slices = std::max<int64_t>(1, (r + slice - 1) / slice);
      const int64_t tm = (m + c.m - 1) / c.m, tn = (n + c.n - 1) / c.n;
      for (const int64_t want : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64}) {
        // the splits' join, and the bias's gradient, which the wide tiles leave to launches of its own
        const double join = (want > 1 ? 4.0 + (double)want * (double)m * (double)n * 8.0 / 6e6 : 0.0) +
                            (bias && c.m == 256 ? 10.0 : 0.0);
        if (want > slices || join >= least) break;
        const int64_t each = (slices + want - 1) / want, parts = (slices + each - 1) / each;
        const double busy = (double)((tm * tn * parts + 255) / 256);
        const double time = join + std::max(c.least, c.first + c.each * busy) * (double)each;
        if (time >= least) continue;
        least = time, tile = c, tiles_m = (int)tm, tiles_n = (int)tn, chunk = each * slice, splits = (int)parts;
      }
    };
    if (!packed) consider(mixed_tile(type));
    else
      for (const auto& c : kPackedTiles) consider(c);
    if (p == kForward && packed && r % 128 == 0)
      for (const auto& c : kDirectTiles) consider(c);
    ldp = (n + 3) / 4 * 4;
    partial_bytes = splits > 1 ? (size_t)splits * m * ldp * sizeof(float) : 0;
    bias_bytes = bias ? (size_t)(wide() ? sum_slabs(r) : (int64_t)splits) * m * sizeof(float) : 0;
  }
  size_t bytes() const { return (partial_bytes + 255) / 256 * 256 + bias_bytes; }
};

template <Product P>
int run_mixed(const char* what, MixedArgs g, int32_t type, void* workspace, size_t workspace_bytes,
              hipStream_t s) {
  const MixedPlan plan(P, g.m, g.n, g.r, type, g.bias_grad != nullptr);
  JN_REQUIRE(!plan.tile.direct || (reinterpret_cast<uintptr_t>(g.scales) & 3) == 0, kInvalidArgument,
             "%s: weight scales must start on 4 bytes", what);
  JN_REQUIRE(!plan.packed || aligned16(g.a), kInvalidArgument, "%s: the operand must start on 16 bytes", what);
  JN_REQUIRE(plan.bytes() == 0 || (workspace && aligned16(workspace) && workspace_bytes >= plan.bytes()),
             kWorkspaceTooSmall, "%s: needs %zu workspace bytes on a 16-byte address, got %zu", what, plan.bytes(),
             workspace_bytes);
  const int64_t threads =  // of the launch that joins the sums
      (plan.partial_bytes ? g.m * (plan.ldp / 4) : 0) + (g.bias_grad && !plan.wide() ? g.m : 0);
  JN_REQUIRE(fits_grid((int64_t)plan.tiles_m * plan.tiles_n * plan.splits, plan.wide() ? 512 : 256) &&
                 fits_grid((threads + 255) / 256, 256),
             kUnsupported, "%s: too many outputs for a launch (%lld x %lld)", what, (long long)g.m, (long long)g.n);
  void* const out = g.out;
  g.tiles_m = plan.tiles_m, g.tiles_n = plan.tiles_n, g.chunk = plan.chunk, g.ldp = plan.ldp;
  const int64_t along = P == kForward ? g.r : g.n;
  g.runs = mx_runs(along), g.pitch = mx_pitch(along, P == kWeightGrad ? kE4m3 : kE2m1);
  if (plan.partial_bytes) g.out = nullptr, g.partial = static_cast<float*>(workspace);
  if (g.bias_grad)
    g.bias_partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + (plan.partial_bytes + 255) / 256 * 256);
  const dim3 grid((unsigned)((int64_t)plan.tiles_m * plan.tiles_n * plan.splits));
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (plan.wide() && g.bias_grad) {  // (the wide tiles have no registers for them)
      if (const int rc = launch_column_sums<T>(g.a, g.r, g.m, g.bias_partial, g.bias_grad, s)) return rc;
      g.bias_grad = nullptr, g.bias_partial = nullptr;
    }
    {
      JN_PROFILE(P == kForward ? "mx_forward_kernel"
                 : P == kInputGrad ? "mx_input_grad_kernel"
                 : P == kWeightGrad ? "mx_weight_grad_kernel"
                                    : "linear_input_grad_kernel",
                 s);
      if (plan.wide()) {
        hipLaunchKernelGGL((mx_bf16_kernel<P, 256, 256, 2, 4, 1>), grid, dim3(512), 0, s, g);
      } else if (!plan.packed) {
        if constexpr (P != kPlainGrad)  // (whose callers ask whether it fits)
          hipLaunchKernelGGL((mx_mixed_kernel<T, P, 128, 128, 2, 2>), grid, dim3(256), 0, s, g);
      } else if (plan.tile.direct) {
        if constexpr (P == kForward) {
          if (plan.tile.m == 128) hipLaunchKernelGGL((mx_direct_kernel<128, 64, 2>), grid, dim3(256), 0, s, g);
          else hipLaunchKernelGGL((mx_direct_kernel<64, 64, 3>), grid, dim3(256), 0, s, g);
        }
      } else if (plan.tile.n == 128) {
        hipLaunchKernelGGL((mx_bf16_kernel<P, 128, 128, 2, 2, 2>), grid, dim3(256), 0, s, g);
      } else if (plan.tile.m == 128) {
        hipLaunchKernelGGL((mx_bf16_kernel<P, 128, 64, 2, 2, 2>), grid, dim3(256), 0, s, g);
      } else {
        hipLaunchKernelGGL((mx_bf16_kernel<P, 64, 64, 2, 2, 2>), grid, dim3(256), 0, s, g);
      }
      JN_LAUNCH_CHECK();
    }
    if (g.partial || g.bias_partial) {
      JN_PROFILE("mx_sum_kernel", s);
      g.out = out;
      hipLaunchKernelGGL(mx_sum_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, g, plan.splits);
      JN_LAUNCH_CHECK();
    }
    return kOk;
  });
}

// ---- forward: microscaled by microscaled --------------------------------------
// v_mfma_scale_f32_16x16x128_f8f6f4 on e2m1 by e2m1: four runs of k an instruction,
// their scales a byte a lane.  A run's products span eight bits, so its sum is exact,
// and the runs' sums are added in fp32.  (With e4m3 the instruction drops what lies
// 14 bits below the run's largest product; x is e2m1 here or not microscaled at all.)
struct LinearArgs {
  const uint8_t* x;   // [m][x_pitch], rows padded with zeros to whole steps
  const uint8_t* xs;  // [m][x_runs]
  const uint8_t* w;   // [n][pitch]
  const uint8_t* ws;  // [n][x_runs]
  const void* bias;   // [n] or null
  void* y;            // [m][n]
  int64_t m, n, x_runs, pitch, x_pitch;
  int tiles_m, tiles_n;
};

constexpr int kStepRuns = 8, kStepBytes = 128;  // of a row in a step of 256 k: a cache line of codes

// Rows of 8 chunks of 16 bytes, permuted so that the 16 lanes of a read that are served
// together (0-3, 12-15 and 20-27 of the first 32, and so on) fall on all 64 banks.
__device__ __forceinline__ int lds_row(int row, int chunk) { return row * 128 + ((chunk ^ (row >> 1)) & 7) * 16; }

// An e2m1 operand: four of the instruction's eight words.
__device__ __forceinline__ intx8 wide(u32x4_nt v) { return intx8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

// Tiles of TM x TN over WM x WN waves in steps of 256 k, LDS double buffered: a step's
// loads go there directly while the step before is multiplied.  Rows past the operands'
// ends are their last rows (their outputs are not written); past a row's end x is zeros,
// so that W may be anything finite there.
// 8,192 cubed takes 321 us (3,425 TFLOP/s, near what the card sustains on random data),
// 8,192 x 2,048 x 16,384 bf16 205 (2,680): eight steps a tile, and its outputs' way out, 256
// KB of fp32 sums rounded through LDS, has no products of another tile beside it (256 x 256
// takes all 256 registers and keeps two more in scratch; a loop over tiles in one workgroup
// had many more there, and was slower).
template <typename T, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM* WN* kWave, 2) void mx_linear_kernel(LinearArgs g) {
  constexpr int WAVES = WM * WN;
  constexpr int MT = TM / WM / 16, NT = TN / WN / 16;          // 16-wide tiles of a wave
  constexpr int XU = TM / (8 * WAVES), WU = TN / (8 * WAVES);  // 16-byte loads a lane and step, eight rows each
  constexpr int kX = TM * kStepBytes, kW = TN * kStepBytes;
  constexpr int kXS = TM * kStepRuns, kWS = TN * kStepRuns;
  constexpr int kStage = kX + kW + kXS + kWS;
  constexpr int kXSL = kXS / 256, kWSL = kWS / 256;            // 4-byte loads of the scales
  static_assert(WAVES % kXSL == 0 && WAVES % kWSL == 0, "a wave loads scales once");
  __shared__ __align__(16) uint8_t smem[2 * kStage];

  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
  const int grp = lane >> 4, col = lane & 15;
  const int wm = wave / WN, wn = wave % WN;
  const TilePlace at(g.tiles_m, g.tiles_n);
  const int64_t m0 = (int64_t)at.mi * TM, n0 = (int64_t)at.ni * TN;
  const int mrows = (int)min((int64_t)TM, g.m - m0), nrows = (int)min((int64_t)TN, g.n - n0);

  // the lane's chunk of its row is the one that belongs in its place
  uint32_t ox[XU], ow[WU];
#pragma unroll
  for (int u = 0; u < XU; ++u) {
    const int row = (u * WAVES + wave) * 8 + lane / 8;
    ox[u] = __umul24(min(row, mrows - 1), (uint32_t)g.x_pitch) + ((lane ^ (row >> 1)) & 7) * 16;
  }
#pragma unroll
  for (int u = 0; u < WU; ++u) {
    const int row = (u * WAVES + wave) * 8 + lane / 8;
    ow[u] = __umul24(min(row, nrows - 1), (uint32_t)g.pitch) + ((lane ^ (row >> 1)) & 7) * 16;
  }
  const int xsrow = tid / 2 % TM, wsrow = tid / 2 % TN;
  const uint32_t oxs = __umul24(min(xsrow, mrows - 1), (uint32_t)g.x_runs) + tid % 2 * 4;
  const uint32_t ows = __umul24(min(wsrow, nrows - 1), (uint32_t)g.x_runs) + tid % 2 * 4;

  const uint32_t lds = lds_offset(smem);
  // The step is in the resources' bases, since a scalar offset is no part of the range
  // check; past the last step all is out of range, which reads nothing (without a branch
  // the loop below is one block).
  const int steps = (int)(g.x_runs / kStepRuns);
  auto load = [&](int step, uint32_t stage) {
    const auto at_step = [&](const uint8_t* rows, int64_t bytes, int each) {
      const int64_t k = (int64_t)step * each;
      return rows_rsrc(rows + k, step < steps ? bytes - k : 0);
    };
    const auto rx = at_step(g.x + m0 * g.x_pitch, (g.m - m0) * g.x_pitch, kStepBytes);
    const auto rw = at_step(g.w + n0 * g.pitch, (g.n - n0) * g.pitch, kStepBytes);
    const auto rxs = at_step(g.xs + m0 * g.x_runs, (g.m - m0) * g.x_runs, kStepRuns);
    const auto rws = at_step(g.ws + n0 * g.x_runs, (g.n - n0) * g.x_runs, kStepRuns);
#pragma unroll
    for (int u = 0; u < XU; ++u) load_lds<16>(rx, lds + stage + (u * WAVES + wave) * 1024, ox[u]);
#pragma unroll
    for (int u = 0; u < WU; ++u) load_lds<16>(rw, lds + stage + kX + (u * WAVES + wave) * 1024, ow[u]);
    load_lds<4>(rxs, lds + stage + kX + kW + wave % kXSL * 256, oxs);
    load_lds<4>(rws, lds + stage + kX + kW + kXS + wave % kWSL * 256, ows);
  };

  floatx4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  // one half step's operands; a lane has the run 4 k + grp of its rows
  u32x4_nt x[MT], w[NT];
  int xs[MT], ws[NT];
  // (a tile's rows are sixteen further on, where the chunks are permuted alike, and the
  // other half step's chunks four: one address an operand, and constants)
  const int xat = lds_row(wm * (TM / WM) + col, grp), wat = kX + lds_row(wn * (TN / WN) + col, grp);
  const int xsat = kX + kW + (wm * (TM / WM) + col) * kStepRuns + grp;
  const int wsat = kX + kW + kXS + (wn * (TN / WN) + col) * kStepRuns + grp;
  auto read_x = [&](uint32_t stage, int k, int j) {
    x[j] = *reinterpret_cast<const u32x4_nt*>(smem + stage + (xat ^ (64 * k)) + j * 16 * kStepBytes);
    xs[j] = smem[stage + xsat + 4 * k + j * 16 * kStepRuns];
  };
  auto read_w = [&](uint32_t stage, int k, int i) {
    w[i] = *reinterpret_cast<const u32x4_nt*>(smem + stage + (wat ^ (64 * k)) + i * 16 * kStepBytes);
    ws[i] = smem[stage + wsat + 4 * k + i * 16 * kStepRuns];
  };
  // A half step's products.  An operand is read anew, for the half step after (from `next`),
  // as soon as its last product is under way; `then` follows the first row of products.
  auto half = [&](uint32_t next, int k, auto then) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[i]), wide(x[j]), acc[i][j], 4, 4, 0, ws[i], 0,
                                                                     xs[j]);
        if (i == NT - 1) {
          read_x(next, k, j);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (i == 0) then();
      read_w(next, k, i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  load(0, 0);
  wait_loads();
  __builtin_amdgcn_s_barrier();
  load(1, kStage);
#pragma unroll
  for (int j = 0; j < MT; ++j) read_x(0, 0, j);
#pragma unroll
  for (int i = 0; i < NT; ++i) read_w(0, 0, i);
  for (int s = 0; s < steps; ++s) {
    const uint32_t cur = (s & 1) * kStage;
    half(cur, 1, [] {});
    // (the last step reads on into the other stage, for nothing)
    half(kStage - cur, 0, [&] {
      // the next step has landed, and every wave has all of this one's operands in
      // registers: its stage is free for the step after the next
      wait_loads();
      __builtin_amdgcn_s_barrier();
      load(s + 2, cur);
    });
  }

  constexpr int kWaveBytes = 2 * kStage / WAVES, GROUP = MT < 4 ? MT : 4;
  static_assert(GROUP * 16 * kLineBytes<T, NT> <= kWaveBytes, "a wave's part of LDS");
  wait_loads();     // those past the last step too:
  __syncthreads();  // LDS is used anew
  store_tile<T, MT, NT, GROUP>(acc, smem + wave * kWaveBytes, static_cast<const T*>(g.bias), static_cast<T*>(g.y),
                               m0 + wm * (TM / WM), n0 + wn * (TN / WN), g.m, g.n, lane);
}

// W's scales with rows of whole steps, 2^0 past their ends: for weights whose rows are not.
__global__ __launch_bounds__(256) void mx_pad_scales_kernel(const uint8_t* scales, int64_t rows, int64_t runs,
                                                            int64_t padded, uint8_t* out) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t words = padded / 4, row = id / words, run = (id - row * words) * 4;
  if (row >= rows) return;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (run + i < runs ? (uint32_t)scales[row * runs + run + i] : 127u) << (8 * i);
  reinterpret_cast<uint32_t*>(out)[id] = w;
}

// ---- forward of few rows --------------------------------------------------------
// Up to 64 rows of x read W once: a workgroup takes NT tiles of sixteen outputs, its
// waves every WAVES-th step of 128 k, straight from memory into registers (a lane has a
// run of 32 k of its row of W, and the same run of its rows of x); their sums join in
// LDS in order.  FORM e2m1: a lane microscales its run of x itself.  Plain x: W's run is
// four bf16 operands of eight, x's as many of each of its terms.  One row by 2,048 x 16,384
// 9 us (17.8 MB of weights, 2 TB/s: a launch, two steps' latency and the join), 64 fp32 rows
// by 512 x 2,048 7 us.
struct RowsArgs {
  const void* x;      // [m][dim]
  const uint8_t* w;   // [n][pitch]
  const uint8_t* ws;  // [n][runs]
  const void* bias;   // [n] or null
  void* y;            // [m][n]
  int64_t m, n, dim, runs, pitch;
};

template <typename T, bool SCALED, int MT, int NT, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void mx_rows_kernel(RowsArgs g) {
  __shared__ __align__(16) float sums[WAVES][NT * MT][256];
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
  const int grp = lane >> 4, col = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * NT * 16, m0 = (int64_t)blockIdx.y * MT * 16;
  const T* x = static_cast<const T*>(g.x);
  constexpr int TERMS = kTerms<T>;

  floatx4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int64_t steps = (g.runs + 3) / 4;
#pragma unroll 2
  for (int64_t s = wave; s < steps; s += WAVES) {
    const int64_t run = s * 4 + grp;
    u32x4_nt w[NT];
    int ws[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int64_t n = min(n0 + i * 16 + col, g.n - 1);  // (past the end: the last row, not written)
      w[i] = u32x4_nt{0, 0, 0, 0}, ws[i] = 127;
      if (run < g.runs) {
        w[i] = *reinterpret_cast<const u32x4_nt*>(g.w + n * g.pitch + run * 16);
        ws[i] = g.ws[n * g.runs + run];
      }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int64_t m = m0 + j * 16 + col, e = run * kMxRun;
      Eight<T> v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q].load(x + m * g.dim + e + q * 8, m < g.m ? g.dim - e - q * 8 : 0);
      if constexpr (SCALED) {
        uint32_t most = 0;
#pragma unroll
        for (int q = 0; q < 32; ++q) most = max(most, __float_as_uint((float)v[q / 8].v[q % 8]) & 0x7FFFFFFFu);
        const int xs = mx_scale_code<kE2m1>(most);
        const float inv = __uint_as_float((uint32_t)(254 - min(xs, 253)) << 23);
        u32x4_nt c;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float f[8];
#pragma unroll
          for (int t = 0; t < 8; ++t) f[t] = (float)v[q].v[t] * inv;
          c[q] = xs == 255 ? 0u : e2m1_word(f);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[i]), wide(c), acc[i][j], 4, 4, 0, ws[i], 0, xs);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          bf16x8v xt[TERMS];
          if constexpr (TERMS == 1) {
            xt[0] = v[q].v;
          } else {
            uint32_t t[4][TERMS];
#pragma unroll
            for (int p = 0; p < 4; ++p) split_pair<T>((float)v[q].v[2 * p], (float)v[q].v[2 * p + 1], t[p]);
#pragma unroll
            for (int p = 0; p < TERMS; ++p)
              xt[p] = __builtin_bit_cast(bf16x8v, make_uint4(t[0][p], t[1][p], t[2][p], t[3][p]));
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const float scale = mx_scale(ws[i]);
            const bf16x8v wt = __builtin_bit_cast(
                bf16x8v, make_uint4(decode_pair<kE2m1, 0>(w[i][q], scale), decode_pair<kE2m1, 1>(w[i][q], scale),
                                    decode_pair<kE2m1, 2>(w[i][q], scale), decode_pair<kE2m1, 3>(w[i][q], scale)));
#pragma unroll
            for (int p = TERMS - 1; p >= 0; --p)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wt, xt[p], acc[i][j], 0, 0, 0);
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<floatx4*>(&sums[wave][i * MT + j][col * 16 + grp * 4]) = acc[i][j];
  __syncthreads();
  for (int id = tid; id < NT * MT * 256; id += WAVES * kWave) {  // [m][n] of the workgroup's outputs
    const int c = id % (NT * 16), row = id / (NT * 16);
    const int64_t n = n0 + c, m = m0 + row;
    if (m >= g.m || n >= g.n) continue;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) t += sums[w][(c / 16) * MT + row / 16][(row % 16) * 16 + c % 16];
    if (g.bias) t += (float)static_cast<const T*>(g.bias)[n];
    static_cast<T*>(g.y)[m * g.n + n] = (T)t;
  }
}

template <typename T, bool SCALED, int MT, int NT>
int launch_rows(const RowsArgs& g, hipStream_t s) {
  const dim3 grid((unsigned)((g.n + NT * 16 - 1) / (NT * 16)), (unsigned)((g.m + MT * 16 - 1) / (MT * 16)));
  JN_PROFILE("mx_rows_kernel", s);
  if (g.runs > 16) hipLaunchKernelGGL((mx_rows_kernel<T, SCALED, MT, NT, 8>), grid, dim3(8 * kWave), 0, s, g);
  else hipLaunchKernelGGL((mx_rows_kernel<T, SCALED, MT, NT, 4>), grid, dim3(4 * kWave), 0, s, g);
  JN_LAUNCH_CHECK();
  return kOk;
}

// Tiles of outputs a workgroup, and tiles of rows.  x's way into registers is the most of
// the work of many rows, so four tiles of outputs share it from 640 on, when that leaves 160
// workgroups.  us with one tile and with four, over 2,048 (bf16 unless said):
//   rows              8,192 outputs  12,000         16,000         16,384
//   1                 4.9 and 6.9    6.6 and 7.0    7.8 and 7.5    7.8 and 7.4
//   16                7.4 and 7.8    10.0 and 7.9   12.6 and 8.2   12.6 and 8.2
//   32                10.9 and 9.9   15.4 and 10.1  19.8 and 10.3  19.8 and 10.4
//   32, e2m1 by e2m1  12.4 and 10.3  16.2 and 10.5  20.5 and 10.9  20.6 and 10.9
//   64                18.2 and 14.9  26.1 and 15.2  33.8 and 15.4  33.9 and 15.4
//   64 fp32           39.1 and 25.8  53.9 and 26.2  68.5 and 27.7  68.5 and 27.5
// (4,096 outputs: 64 rows 10.3 and 14.9, fp32 20.1 and 25.5, 1 row 4.1 and 6.9.)
constexpr int64_t kShareOuts = 640;
template <typename T, bool SCALED>
int run_rows(const RowsArgs& g, hipStream_t s) {
  const int64_t rows = (g.m + 15) / 16, outs = (g.n + 15) / 16;
  const bool share = outs >= kShareOuts;
  if (rows == 1) return share ? launch_rows<T, SCALED, 1, 4>(g, s) : launch_rows<T, SCALED, 1, 1>(g, s);
  if (share) return rows == 2 ? launch_rows<T, SCALED, 2, 4>(g, s) : launch_rows<T, SCALED, 4, 4>(g, s);
  if (outs >= 256) return rows == 2 ? launch_rows<T, SCALED, 2, 1>(g, s) : launch_rows<T, SCALED, 4, 1>(g, s);
  return rows > 2 && outs >= 128 ? launch_rows<T, SCALED, 2, 1>(g, s) : launch_rows<T, SCALED, 1, 1>(g, s);
}

// Few rows: microscaling x apart costs more than it does here until it is shared by
// more workgroups (bf16, 2,048 x 16,384, both e2m1: 32 rows 11.0 us here, 64 in two launches
// 11.0).  x as it is: 64 rows 15.4 us here, 65 in tiles 18.4.
bool few_rows(int64_t rows, int32_t activations) { return rows <= (activations == kPlain ? 64 : 32); }

// x microscaled for this product: rows of whole steps.
int64_t step_runs(int64_t dim) { return (mx_runs(dim) + kStepRuns - 1) / kStepRuns * kStepRuns; }
size_t linear_codes_bytes(int64_t rows, int64_t dim) { return (size_t)(rows * step_runs(dim) * 16); }

template <typename T, int TM, int TN, int WM, int WN>
int launch_linear(LinearArgs g, hipStream_t s) {
  g.tiles_m = (int)((g.m + TM - 1) / TM), g.tiles_n = (int)((g.n + TN - 1) / TN);
  JN_PROFILE("mx_linear_kernel", s);
  hipLaunchKernelGGL((mx_linear_kernel<T, TM, TN, WM, WN>), dim3((unsigned)((int64_t)g.tiles_m * g.tiles_n)),
                     dim3(WM * WN * kWave), 0, s, g);
  JN_LAUNCH_CHECK();
  return kOk;
}

int check_product(const char* what, int64_t rows, int64_t dim, int64_t out, int32_t type) {
  JN_REQUIRE(known_type(type), kInvalidArgument, "%s: unknown element type %d", what, type);
  JN_REQUIRE(rows >= 1 && dim >= 1 && out >= 1 && rows < (int64_t(1) << 31) && dim < (int64_t(1) << 24) &&
                 out < (int64_t(1) << 24),
             kInvalidArgument, "%s: needs 1 to 2^31 - 1 rows and 1 to 2^24 - 1 inputs and outputs, got %lld, %lld, %lld",
             what, (long long)rows, (long long)dim, (long long)out);
  return kOk;
}

}  // namespace
}  // namespace jakal

using namespace jakal;

extern "C" {

size_t jn_mx_linear_forward_workspace_bytes(int64_t rows, int64_t dim, int64_t out, int32_t type, int32_t activations) {
  if (check_product("mx_linear", rows, dim, out, type) || few_rows(rows, activations)) return 0;
  if (activations == kPlain) return MixedPlan(kForward, rows, out, dim, type, false).bytes();
  return linear_codes_bytes(rows, dim) + (size_t)((rows + (mx_runs(dim) % kStepRuns ? out : 0)) * step_runs(dim));
}

int jn_mx_linear_forward(const void* x, const void* weight_codes, const void* weight_scales, const void* bias,
                         int64_t rows, int64_t dim, int64_t out, int32_t type, int32_t activations, void* y,
                         void* workspace, size_t workspace_bytes, jn_stream_t stream) {
  if (const int rc = check_product("mx_linear", rows, dim, out, type)) return rc;
  JN_REQUIRE(activations == kE2m1 || activations == kPlain, kInvalidArgument,
             "mx_linear: activations are e2m1 (1) or as they are (-1), got %d", activations);
  JN_REQUIRE(x && weight_codes && weight_scales && y, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(aligned16(weight_codes) && aligned16(y), kInvalidArgument,
             "mx_linear: weight codes and outputs must start on 16 bytes");
  const auto s = static_cast<hipStream_t>(stream);
  if (few_rows(rows, activations)) {
    RowsArgs g{};
    g.x = x, g.w = static_cast<const uint8_t*>(weight_codes), g.ws = static_cast<const uint8_t*>(weight_scales);
    g.bias = bias, g.y = y, g.m = rows, g.n = out, g.dim = dim, g.runs = mx_runs(dim), g.pitch = mx_pitch(dim, kE2m1);
    return with_type(type, [&](auto* t) -> int {
      using T = std::remove_pointer_t<decltype(t)>;
      return activations == kPlain ? run_rows<T, false>(g, s) : run_rows<T, true>(g, s);
    });
  }
  if (activations == kPlain) {
    MixedArgs g{};
    g.a = x, g.codes = static_cast<const uint8_t*>(weight_codes), g.scales = static_cast<const uint8_t*>(weight_scales);
    g.bias = bias, g.out = y, g.m = rows, g.n = out, g.r = dim, g.lda = dim;
    return run_mixed<kForward>("mx_linear", g, type, workspace, workspace_bytes, s);
  }
  const size_t need = jn_mx_linear_forward_workspace_bytes(rows, dim, out, type, activations);
  JN_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, kWorkspaceTooSmall,
             "mx_linear: needs %zu workspace bytes on a 16-byte address, got %zu", need, workspace_bytes);
  JN_REQUIRE((reinterpret_cast<uintptr_t>(weight_scales) & 3) == 0 || mx_runs(dim) % kStepRuns, kInvalidArgument,
             "mx_linear: weight scales must start on 4 bytes");
  LinearArgs g{};
  uint8_t* const codes = static_cast<uint8_t*>(workspace);
  uint8_t* const scales = codes + linear_codes_bytes(rows, dim);
  g.x = codes, g.xs = scales;
  g.w = static_cast<const uint8_t*>(weight_codes), g.ws = static_cast<const uint8_t*>(weight_scales);
  g.bias = bias, g.y = y, g.m = rows, g.n = out, g.pitch = mx_pitch(dim, kE2m1);
  g.x_runs = step_runs(dim), g.x_pitch = g.x_runs * 16;
  // The widest tiles that keep three quarters of the CUs busy (bf16, us with tiles of 256,
  // 128 and 64: 768 x 2,048 x 16,384 28.3, 29.3 and 45.9; 768 x 4,096 x 4,096 38.5, 23.6 and
  // 28.9; 512 x 4,096 x 4,096 37.9, 22.1 and 20.1; 4,096 x 2,048 x 2,048 30.5, 24.8, 36.7).
  const auto tiles = [&](int64_t edge) { return (rows + edge - 1) / edge * ((out + edge - 1) / edge); };
  const int64_t tile = tiles(256) >= 192 ? 256 : tiles(128) >= 192 ? 128 : 64;
  const int64_t words = mx_runs(dim) % kStepRuns ? out * g.x_runs / 4 : 0;  // of W's scales in rows of whole steps
  JN_REQUIRE(fits_grid(tiles(tile), tile == 256 ? 512 : 256) && fits_grid((words + 255) / 256, 256), kUnsupported,
             "mx_linear: too many outputs for a launch (%lld x %lld)", (long long)rows, (long long)out);
  if (words) {
    uint8_t* const padded = scales + rows * g.x_runs;
    JN_PROFILE("mx_pad_scales_kernel", s);
    hipLaunchKernelGGL(mx_pad_scales_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s, g.ws, out,
                       mx_runs(dim), g.x_runs, padded);
    JN_LAUNCH_CHECK();
    g.ws = padded;
  }
  if (const int rc = launch_mx_quantize(x, rows, dim, type, kE2m1, codes, scales, s, g.x_runs)) return rc;
  return with_type(type, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (tile == 256) return launch_linear<T, 256, 256, 2, 4>(g, s);
    if (tile == 128) return launch_linear<T, 128, 128, 2, 2>(g, s);
    return launch_linear<T, 64, 64, 2, 2>(g, s);
  });
}

size_t jn_mx_linear_backward_workspace_bytes(int64_t rows, int64_t dim, int64_t out, int32_t type) {
  if (check_product("mx_linear backward", rows, dim, out, type)) return 0;
  return MixedPlan(kInputGrad, rows, dim, out, type, false).bytes();
}

int jn_mx_linear_backward(const void* grad_y, const void* weight_codes, const void* weight_scales, int64_t rows,
                          int64_t dim, int64_t out, int32_t type, void* grad_x, void* workspace,
                          size_t workspace_bytes, jn_stream_t stream) {
  if (const int rc = check_product("mx_linear backward", rows, dim, out, type)) return rc;
  JN_REQUIRE(grad_y && weight_codes && weight_scales && grad_x, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(aligned16(weight_codes) && aligned16(grad_x), kInvalidArgument,
             "mx_linear backward: weight codes and grad_x must start on 16 bytes");
  MixedArgs g{};
  g.a = grad_y, g.codes = static_cast<const uint8_t*>(weight_codes);
  g.scales = static_cast<const uint8_t*>(weight_scales);
  g.out = grad_x, g.m = rows, g.n = dim, g.r = out, g.lda = out;
  return run_mixed<kInputGrad>("mx_linear backward", g, type, workspace, workspace_bytes,
                        static_cast<hipStream_t>(stream));
}

size_t jn_mx_weight_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t out, int32_t type, int32_t bias) {
  if (check_product("mx_weight_grad", rows, dim, out, type)) return 0;
  return MixedPlan(kWeightGrad, out, dim, rows, type, bias != 0).bytes();
}

int jn_mx_weight_grad(const void* grad_y, const void* codes, const void* scales, int64_t rows, int64_t dim,
                      int64_t out, int32_t type, void* grad_weight, void* grad_bias, void* workspace,
                      size_t workspace_bytes, jn_stream_t stream) {
  if (const int rc = check_product("mx_weight_grad", rows, dim, out, type)) return rc;
  JN_REQUIRE(grad_y && codes && scales && grad_weight, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(aligned16(codes) && aligned16(grad_weight), kInvalidArgument,
             "mx_weight_grad: codes and grad_weight must start on 16 bytes");
  MixedArgs g{};
  g.a = grad_y, g.codes = static_cast<const uint8_t*>(codes), g.scales = static_cast<const uint8_t*>(scales);
  g.out = grad_weight, g.bias_grad = grad_bias, g.m = out, g.n = dim, g.r = rows, g.lda = out;
  return run_mixed<kWeightGrad>("mx_weight_grad", g, type, workspace, workspace_bytes,
                         static_cast<hipStream_t>(stream));
}

int32_t jn_linear_input_grad_fits(int64_t rows, int64_t dim, int64_t out, int32_t type) {
  if (check_product("linear backward", rows, dim, out, type)) return 0;
  // Measured with the library's product (us, here and there, in captured calls; eager, the
  // library's takes the host 12 us more).  Long sums leave most CUs to the splits that the
  // library does not make:
  //   outputs  1 x 2,048      64 x 512      256 x 2,048   1,024 x 2,048  2,048 x 2,048
  //   16,384   23.1 and 36.4  16.1 and 68   33.8 and 65   78 and 112     133 and 144
  //   12,000   21.5 and 26.7  14.6 and 59   30.0 and 56   66 and 90      106 and 117
  //   8,192    18.1 and 14.6  10.6 and 36   23.9 and 35   52 and 58      79 and 76
  //   6,144    14.3 and 10.0  10.3 and 28   20.8 and 27   46 and 44      66 and 59
  //   4,096    16.4 and 7.8   9.7 and 21    21.4 and 20   34 and 32      53 and 42
  //   2,048    10.1 and 6.2   7.8 and 12    15.1 and 12   22 and 19      29 and 24
  //   768      6.9 and 4.5    7.0 and 7.4   7.8 and 7.0   11.0 and 9.7   14.1 and 12.1
  //   512      5.9 and 4.2    6.1 and 6.2   6.3 and 6.9   8.6 and 8.6    11.2 and 11.0
  //   256      4.5 and 3.9    4.6 and 4.9   4.7 and 5.2   6.3 and 6.6    8.1 and 8.3
  // (16,384: 2,048 x 4,096 265 and 245.)  Between 512 and 8,192 outputs the library's is as
  // fast or faster but for tens of rows (from 4,096 on, hundreds), which are left to it too;
  // up to 16,384 the limits are those of 8,192, though 12,000 would bear 16,384's.
  const MixedPlan plan(kPlainGrad, rows, dim, out, type, false);
  const int64_t outputs = rows * dim;
  if (!plan.packed) return 0;
  if (out >= 16384) return outputs <= (1 << 22);
  if (out >= 8192) return rows >= 16 && outputs <= (1 << 21);
  return out <= 512 && rows >= (out <= 256 ? 16 : 64) && outputs <= (1 << 24);
}

size_t jn_linear_input_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t out, int32_t type) {
  if (check_product("linear backward", rows, dim, out, type)) return 0;
  return MixedPlan(kPlainGrad, rows, dim, out, type, false).bytes();
}

int jn_linear_input_grad(const void* grad_y, const void* weight, int64_t rows, int64_t dim, int64_t out, int32_t type,
                         void* grad_x, void* workspace, size_t workspace_bytes, jn_stream_t stream) {
  if (const int rc = check_product("linear backward", rows, dim, out, type)) return rc;
  JN_REQUIRE(grad_y && weight && grad_x, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(aligned16(weight) && aligned16(grad_x), kInvalidArgument,
             "linear backward: weight and grad_x must start on 16 bytes");
  JN_REQUIRE(jn_linear_input_grad_fits(rows, dim, out, type), kUnsupported,
             "linear backward: these sizes are left to a library product");
  MixedArgs g{};
  g.a = grad_y, g.codes = static_cast<const uint8_t*>(weight), g.out = grad_x;
  g.m = rows, g.n = dim, g.r = out, g.lda = out;
  return run_mixed<kPlainGrad>("linear backward", g, type, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

size_t jn_column_sums_workspace_bytes(int64_t rows, int64_t dim) {
  return rows < 1 || dim < 1 ? 0 : (size_t)(sum_slabs(rows) * dim) * sizeof(float);
}

int jn_column_sums(const void* x, int64_t rows, int64_t dim, int32_t type, void* sums, void* workspace,
                   size_t workspace_bytes, jn_stream_t stream) {
  if (const int rc = check_product("column_sums", rows, 1, dim, type)) return rc;
  JN_REQUIRE(x && sums, kInvalidArgument, "null tensor pointer");
  const size_t need = jn_column_sums_workspace_bytes(rows, dim);
  JN_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, kWorkspaceTooSmall,
             "column_sums: needs %zu workspace bytes on a 16-byte address, got %zu", need, workspace_bytes);
  const auto s = static_cast<hipStream_t>(stream);
  return with_type(type, [&](auto* t) -> int {
    return launch_column_sums<std::remove_pointer_t<decltype(t)>>(x, rows, dim, static_cast<float*>(workspace), sums, s);
  });
}

}  // extern "C"
