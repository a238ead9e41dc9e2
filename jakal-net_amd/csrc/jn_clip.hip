// Global norm over many gradient tensors, and clipping (jn_grads_*).
//
//   n = sqrt(sum g^2) or max |g| over every element of every tensor,
//   c = min(1, max_norm / (n + 1e-6)),  out = c g
//
// A launch takes up to kListMax tensors, whose addresses and sizes travel in
// its arguments (no table in device memory, so a captured call carries its
// own).  The elements are cut into chunks that lie in one tensor each; workgroup
// b takes chunks b, b + grid, ..., so that every sum has one fixed order.
// Squares are summed in 64 bits: fp32 elements beyond 2^63 do not overflow, and
// the order of the sum does not show in the norm's fp32 digits.
#include <algorithm>
#include <memory>
#include <new>

#include "../../include/jakal_net_hip.h"
#include "jn_internal.hpp"
#include "jn_rows.hpp"

namespace jakal {
namespace {

constexpr int kClipThreads = 256;
constexpr int kChunk = 8192;         // elements
constexpr int kListMax = 164;        // tensors of one launch (4 KB of kernel arguments)
constexpr int64_t kMaxPartials = 2048;  // shared out over the launches; beyond it one for each further launch

struct TensorList {
  const void* in[kListMax];
  void* out[kListMax];
  int32_t first[kListMax + 1];  // first chunk; behind the last tensor, all chunks
  int32_t last[kListMax];       // elements of the last chunk | type << 16 | output type << 20
  int32_t count;
};
static_assert(sizeof(TensorList) <= 4000, "kernel arguments stay within 4 KB");

struct Chunk {
  int tensor;
  int64_t begin;
  int size, type, out_type;
};

// A chunk's place (a uniform binary search for its tensor).
__device__ __forceinline__ Chunk chunk_at(const TensorList& l, int c) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (l.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  const int meta = l.last[lo];
  return {lo, (int64_t)(c - l.first[lo]) * kChunk, c + 1 == l.first[lo + 1] ? meta & 0xffff : kChunk,
          meta >> 16 & 15, meta >> 20};
}

// max that keeps a NaN
__device__ __forceinline__ double max_nan(double m, double v) { return v > m || v != v ? v : m; }

template <bool MAX>
__device__ __forceinline__ double join(double a, double b) {
  return MAX ? max_nan(a, b) : a + b;
}

template <bool MAX>
__device__ double group_join(double v, double* lds) {
  lds[threadIdx.x] = v;
  for (int step = kClipThreads / 2; step > 0; step /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < step) lds[threadIdx.x] = join<MAX>(lds[threadIdx.x], lds[threadIdx.x + step]);
  }
  __syncthreads();
  return lds[0];
}

// Elements before the first whole pack of W: views of one flat buffer start
// anywhere in it.
template <int W, typename T>
__device__ __forceinline__ int pack_head(const T* p) {
  return (int)((0 - reinterpret_cast<uintptr_t>(p) / sizeof(T)) & (W - 1));
}

// A chunk's part of a norm: 16-byte packs, and single elements on either side.
template <bool MAX, typename T>
__device__ __forceinline__ double chunk_norm(const T* p, int n, double s) {
  constexpr int W = 16 / sizeof(T), kUnroll = kChunk / W / kClipThreads;
  const auto take = [&](float v) {
    const double d = v;
    s = MAX ? max_nan(s, fabs(d)) : s + d * d;
  };
  const int t = threadIdx.x, head = min(pack_head<W>(p), n), packs = (n - head) / W, tail = head + packs * W;
  Raw<T, W> raw[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if (i * kClipThreads + t < packs) raw[i].load(p + head + (i * kClipThreads + t) * W);
  }
  if (t < head) take((float)p[t]);
  if (tail + t < n) take((float)p[tail + t]);
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if (i * kClipThreads + t >= packs) continue;
    float v[W];
    raw[i].unpack(v);
#pragma unroll
    for (int j = 0; j < W; ++j) take(v[j]);
  }
  return s;
}

// Bound by the read: 145 tensors of 45.6M elements, fp32 32 us (182 MB, 5.6 TB/s),
// bf16 20 (91 MB, 4.7).  Chunks of 4,096 and 16,384 elements, and 1,024 workgroups,
// were within 3 %.
template <bool MAX>
__global__ __launch_bounds__(kClipThreads) void grads_norm_kernel(TensorList l, double* partial) {
  __shared__ double lds[kClipThreads];
  double s = 0.0;
  for (int i = blockIdx.x; i < l.first[l.count]; i += gridDim.x) {
    const Chunk c = chunk_at(l, i);
    const void* in = l.in[c.tensor];
    if (c.type == kTypeF32) s = chunk_norm<MAX>(static_cast<const float*>(in) + c.begin, c.size, s);
    else if (c.type == kTypeBf16) s = chunk_norm<MAX>(static_cast<const bf16_t*>(in) + c.begin, c.size, s);
    else s = chunk_norm<MAX>(static_cast<const f16_t*>(in) + c.begin, c.size, s);
  }
  s = group_join<MAX>(s, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

template <bool MAX>
__device__ double total_norm(const double* partial, int n, double* lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kClipThreads) s = join<MAX>(s, partial[i]);
  s = group_join<MAX>(s, lds);
  return MAX ? s : sqrt(s);
}

template <bool MAX>
__global__ __launch_bounds__(kClipThreads) void grads_norm_finish_kernel(const double* partial, int n, float* norm) {
  __shared__ double lds[kClipThreads];
  const double s = total_norm<MAX>(partial, n, lds);
  if (threadIdx.x == 0) *norm = (float)s;
}

// A chunk times the factor, in packs that are 16 bytes of the wider type, so
// that loads and stores both run through memory without gaps; where the two
// tensors' packs do not start at the same element, element by element.
template <bool STREAM, typename TI, typename TO>
__device__ __forceinline__ void chunk_scale(const TI* p, TO* o, int n, float scale) {
  constexpr int W = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
  constexpr int kUnroll = 8;  // packs in flight
  const int t = threadIdx.x, head = min(pack_head<W>(p), n);
  if (pack_head<W>(o) != pack_head<W>(p)) {
#pragma unroll 8
    for (int i = t; i < n; i += kClipThreads) o[i] = (TO)(scale * (float)p[i]);
    return;
  }
  const int packs = (n - head) / W, tail = head + packs * W;
  if (t < head) o[t] = (TO)(scale * (float)p[t]);
  if (tail + t < n) o[tail + t] = (TO)(scale * (float)p[tail + t]);
  p += head, o += head;
  for (int first = t; first < packs; first += kUnroll * kClipThreads) {
    Raw<TI, W> raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int k = first + i * kClipThreads;
      if (k < packs) raw[i].template load<STREAM>(p + k * W);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int k = first + i * kClipThreads;
      if (k >= packs) continue;
      float v[W];
      raw[i].unpack(v);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] *= scale;
      store_raw<TO, W, STREAM>(o + k * W, v);
    }
  }
}

template <bool STREAM, typename TI>
__device__ __forceinline__ void chunk_scale_to(const TI* p, void* out, int64_t begin, int n, int type, float scale) {
  if (type == kTypeF32) chunk_scale<STREAM>(p, static_cast<float*>(out) + begin, n, scale);
  else if (type == kTypeBf16) chunk_scale<STREAM>(p, static_cast<bf16_t*>(out) + begin, n, scale);
  else chunk_scale<STREAM>(p, static_cast<f16_t*>(out) + begin, n, scale);
}

// Every workgroup joins the norm's partials (in one order; partial_count bounds
// them) rather than wait for a launch that does; the first writes the norm.
// 145 tensors of 45.6M elements, fp32 into fp32: 57 us, 365 MB, 6.4 TB/s (with
// ordinary stores 68, and the next norm 47 instead of 32: it has their lines to
// write back); bf16 into fp32 42 us.
template <bool MAX, bool STREAM>
__global__ __launch_bounds__(kClipThreads) void grads_scale_kernel(TensorList l, const double* partial, int n,
                                                                   double max_norm, float* norm) {
  __shared__ double lds[kClipThreads];
  const double total = total_norm<MAX>(partial, n, lds);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const double ratio = max_norm / (total + 1e-6);
  const float scale = ratio < 1.0 || ratio != ratio ? (float)ratio : 1.0f;
  for (int i = blockIdx.x; i < l.first[l.count]; i += gridDim.x) {
    const Chunk c = chunk_at(l, i);
    const void* in = l.in[c.tensor];
    void* out = l.out[c.tensor];
    if (scale == 1.0f && in == out) continue;  // unchanged in place
    if (c.type == kTypeF32)
      chunk_scale_to<STREAM>(static_cast<const float*>(in) + c.begin, out, c.begin, c.size, c.out_type, scale);
    else if (c.type == kTypeBf16)
      chunk_scale_to<STREAM>(static_cast<const bf16_t*>(in) + c.begin, out, c.begin, c.size, c.out_type, scale);
    else
      chunk_scale_to<STREAM>(static_cast<const f16_t*>(in) + c.begin, out, c.begin, c.size, c.out_type, scale);
  }
}

// The tensors of a call in launches of up to kListMax, empty ones left out.
struct ListCursor {
  const void* const* in;
  void* const* out;
  const int64_t* counts;
  const int32_t* types;
  const int32_t* out_types;
  int64_t n, at = 0;

  bool next(TensorList& l) {
    l.count = l.first[0] = 0;
    for (; at < n && l.count < kListMax; ++at) {
      const int64_t chunks = (counts[at] + kChunk - 1) / kChunk;
      if (chunks == 0) continue;
      l.in[l.count] = in[at];
      l.out[l.count] = out ? out[at] : nullptr;
      l.last[l.count] =
          (int32_t)(counts[at] - (chunks - 1) * kChunk) | types[at] << 16 | (out ? out_types[at] : 0) << 20;
      l.first[l.count + 1] = l.first[l.count] + (int32_t)chunks;
      ++l.count;
    }
    return l.count > 0;
  }
};

int check_list(const void* const* in, void* const* out, const int64_t* counts, const int32_t* types,
               const int32_t* out_types, int64_t n, int32_t norm_kind, bool clip) {
  JN_REQUIRE(n >= 0 && n < (1LL << 28) && (n == 0 || (in && counts && types && (!clip || (out && out_types)))),
             kInvalidArgument, "a list of up to 2^28 tensors, none of its arrays null");
  JN_REQUIRE(norm_kind == 0 || norm_kind == 1, kInvalidArgument, "the norm is 0 (Euclidean) or 1 (maximum), got %d",
             (int)norm_kind);
  int64_t chunks = 0;
  for (int64_t i = 0; i < n; ++i) {
    JN_REQUIRE(counts[i] >= 0 && counts[i] < (1LL << 40), kInvalidArgument,
               "tensor %lld: sizes are 0 to 2^40 - 1 elements, got %lld", (long long)i, (long long)counts[i]);
    JN_REQUIRE(known_type(types[i]) && (!clip || known_type(out_types[i])), kInvalidArgument,
               "tensor %lld: element types are 0 (fp32), 1 (bf16) and 2 (fp16)", (long long)i);
    JN_REQUIRE(counts[i] == 0 || (in[i] && (!clip || out[i])), kInvalidArgument, "tensor %lld: null pointer",
               (long long)i);
    JN_REQUIRE(!clip || counts[i] == 0 || in[i] != out[i] || types[i] == out_types[i], kInvalidArgument,
               "tensor %lld: in place its element type stays", (long long)i);
    chunks += (counts[i] + kChunk - 1) / kChunk;
    JN_REQUIRE(chunks < (1LL << 31), kUnsupported, "at most 2^44 elements in all");
  }
  return kOk;
}

// No output may meet another tensor's memory: workgroups read and write the
// list in no order.  (In place, the pair is one span.)
int check_apart(const void* const* in, void* const* out, const int64_t* counts, const int32_t* types,
                const int32_t* out_types, int64_t n) {
  struct Span {
    uintptr_t begin, end;
    bool write;
  };
  const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[2 * n + 1]);
  JN_REQUIRE(spans, kUnsupported, "no host memory for a list of %lld tensors", (long long)n);
  Span* end = spans.get();
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    const auto r = reinterpret_cast<uintptr_t>(in[i]), w = reinterpret_cast<uintptr_t>(out[i]);
    *end++ = {w, w + (uintptr_t)counts[i] * type_bytes(out_types[i]), true};
    if (r != w) *end++ = {r, r + (uintptr_t)counts[i] * type_bytes(types[i]), false};
  }
  std::sort(spans.get(), end, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;  // the farthest ends so far
  for (const Span* at = spans.get(); at != end; ++at) {
    const Span& s = *at;
    JN_REQUIRE(s.begin >= (s.write ? any : written), kInvalidArgument,
               "an output shares memory with another tensor of the lists");
    any = std::max(any, s.end);
    if (s.write) written = std::max(written, s.end);
  }
  return kOk;
}

int64_t total_chunks(const int64_t* counts, int64_t n) {
  int64_t s = 0;
  for (int64_t i = 0; i < n; ++i) s += (counts[i] + kChunk - 1) / kChunk;
  return s;
}

// Workgroups of a launch, a partial each: its share of kMaxPartials rounded
// down, and one at least.
int list_groups(const TensorList& l, int64_t total) {
  const int64_t chunks = l.first[l.count];
  return (int)(total <= kMaxPartials ? chunks : std::max<int64_t>(1, chunks * kMaxPartials / total));
}

// The most partials that a list of n tensors leaves: the shares come to
// kMaxPartials, and launches whose share is none add one each.
int64_t partial_count(int64_t n) { return kMaxPartials + n / kListMax + 1; }

template <bool MAX>
int launch_partials(ListCursor c, int64_t total, double* partial, int* found, hipStream_t s) {
  TensorList l;
  *found = 0;
  while (c.next(l)) {
    const int groups = list_groups(l, total);
    JN_PROFILE("grads_norm_kernel", s);
    hipLaunchKernelGGL(grads_norm_kernel<MAX>, dim3(groups), dim3(kClipThreads), 0, s, l, partial + *found);
    JN_LAUNCH_CHECK();
    *found += groups;
  }
  return kOk;
}

template <bool MAX>
int launch_clip(ListCursor c, int64_t total, double max_norm, float* norm, double* partial, bool clip,
                hipStream_t s) {
  int found = 0;
  if (const int rc = launch_partials<MAX>(c, total, partial, &found, s)) return rc;
  TensorList l;
  if (!clip || !c.next(l)) {
    JN_PROFILE("grads_norm_finish_kernel", s);
    hipLaunchKernelGGL(grads_norm_finish_kernel<MAX>, dim3(1), dim3(kClipThreads), 0, s, partial, found, norm);
    JN_LAUNCH_CHECK();
    return kOk;
  }
  // What is read and written (in place: written where it was read).  Beyond the
  // cache it streams.  fp32 into fp32, streaming and with ordinary accesses, alone
  // and with a fused AdamW over the outputs behind it: 256 MB 72 and 73, 665 and
  // 683 us; 365 MB 97 and 105, 737 and 757; 512 MB 133 and 165, 839 and 865; in
  // place 365 MB 85 and 87, 872 and 878.  (A pass that does nothing but read the
  // outputs behind it finds more of them after ordinary accesses up to 384 MB:
  // 256 MB 121 and 107, 384 MB 176 and 178, 512 MB 232 and 245.)
  int64_t bytes = 0;
  for (int64_t i = 0; i < c.n; ++i)
    bytes += c.counts[i] * (type_bytes(c.types[i]) + (c.in[i] == c.out[i] ? 0 : type_bytes(c.out_types[i])));
  const auto kernel = bytes > kCacheBytes ? grads_scale_kernel<MAX, true> : grads_scale_kernel<MAX, false>;
  do {
    JN_PROFILE("grads_scale_kernel", s);
    hipLaunchKernelGGL(kernel, dim3(list_groups(l, total)), dim3(kClipThreads), 0, s, l, partial, found, max_norm,
                       norm);
    JN_LAUNCH_CHECK();
    norm = nullptr;
  } while (c.next(l));
  return kOk;
}

}  // namespace
}  // namespace jakal

using namespace jakal;

extern "C" {

size_t jn_grads_workspace_bytes(int64_t tensors) {
  return tensors < 0 ? 0 : (size_t)partial_count(tensors) * sizeof(double);
}

int jn_grads_norm(const void* const* grads, const int64_t* counts, const int32_t* types, int64_t tensors,
                  int32_t norm_kind, float* norm, void* workspace, size_t workspace_bytes, jn_stream_t stream) {
  if (const int rc = check_list(grads, nullptr, counts, types, nullptr, tensors, norm_kind, false)) return rc;
  JN_REQUIRE(norm && workspace, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(workspace_bytes >= jn_grads_workspace_bytes(tensors), kWorkspaceTooSmall,
             "gradient norm needs %zu workspace bytes, got %zu", jn_grads_workspace_bytes(tensors), workspace_bytes);
  const ListCursor c{grads, nullptr, counts, types, nullptr, tensors};
  const auto run = norm_kind ? launch_clip<true> : launch_clip<false>;
  return run(c, total_chunks(counts, tensors), 0.0, norm, static_cast<double*>(workspace), false,
             static_cast<hipStream_t>(stream));
}

int jn_grads_clip(const void* const* grads, void* const* out, const int64_t* counts, const int32_t* types,
                  const int32_t* out_types, int64_t tensors, double max_norm, int32_t norm_kind, float* norm,
                  void* workspace, size_t workspace_bytes, jn_stream_t stream) {
  if (const int rc = check_list(grads, out, counts, types, out_types, tensors, norm_kind, true)) return rc;
  if (const int rc = check_apart(grads, out, counts, types, out_types, tensors)) return rc;
  JN_REQUIRE(max_norm >= 0.0, kInvalidArgument, "max_norm must not be negative");
  JN_REQUIRE(norm && workspace, kInvalidArgument, "null tensor pointer");
  JN_REQUIRE(workspace_bytes >= jn_grads_workspace_bytes(tensors), kWorkspaceTooSmall,
             "gradient clipping needs %zu workspace bytes, got %zu", jn_grads_workspace_bytes(tensors),
             workspace_bytes);
  const ListCursor c{grads, out, counts, types, out_types, tensors};
  const auto run = norm_kind ? launch_clip<true> : launch_clip<false>;
  return run(c, total_chunks(counts, tensors), max_norm, norm, static_cast<double*>(workspace), true,
             static_cast<hipStream_t>(stream));
}

}  // extern "C"
