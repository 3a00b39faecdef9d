// Global norm of a list of gradient tensors, and clipping by it:
//   norm = scale * sqrt(sum_t sum_j g_t[j]^2)        factor = limit / max(norm, limit)
//   out_t[j] = g_t[j] * (scale * factor)              (NaN everywhere when the norm is not finite)
// which is what a step needs between its backward pass and its update when the gradient may not be longer than `limit`.
//
// The values are squared and summed in fp64: a square of any fp32 value is representable there (fp32 squares overflow
// from 1.8e19 on and vanish below 1e-23), and the sum over 1e9 values keeps all digits the result has.  The fp64 units
// keep up with memory: one conversion and one fma per value.  No atomics: a workgroup adds up its chunks in a fixed
// order and leaves one partial sum, and every workgroup of the second pass adds all partial sums in the same order, so
// the result is bitwise reproducible and no third launch is needed between the two passes.
//
// Bound by memory: the first pass reads every gradient, the second reads it again and writes it.  The second pass walks
// the chunks in the opposite order, so that what the first one read last is found in the 256 MB memory-side cache.
#include "common.hpp"
#include "api.h"

namespace dtf {

constexpr int kSpans = 72;          // spans per launch: the table travels as a kernel argument (4 KB limit), so a captured
                                    // launch carries it and no upload or device table exists
constexpr int kClipThreads = 256;
constexpr int kClipVec = kClipThreads * 16;   // bytes one workgroup reads per load instruction

struct ClipBatch {
  DtfClipSpan s[kSpans];
  int chunk_end[kSpans];            // running number of chunks up to and including span k
  int count;
  int chunks;                       // == chunk_end[count - 1]
  int chunk_bytes;                  // of the input, a multiple of kClipVec
};
static_assert(sizeof(ClipBatch) + 64 <= 4096, "kernel arguments");

// 16 bytes at any element alignment (global memory takes unaligned vector accesses; a tensor of an arena may start at
// any element)
typedef u32x4 u32x4_any __attribute__((aligned(2)));
__device__ __forceinline__ u32x4 load_any(const void* p) {
  const u32x4 v = *reinterpret_cast<const u32x4_any*>(p);
  return v;
}
__device__ __forceinline__ void store_any(void* p, u32x4 v) { *reinterpret_cast<u32x4_any*>(p) = v; }

__device__ __forceinline__ void unpack(const float*, const u32x4& v, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned w = v[i];        // (a bit_cast of the vector element itself reads element 0)
    f[i] = __builtin_bit_cast(float, w);
  }
}
__device__ __forceinline__ void unpack(const bf16*, const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned lo = v[i] << 16, hi = v[i] & 0xffff0000u;
    f[2 * i] = __builtin_bit_cast(float, lo);
    f[2 * i + 1] = __builtin_bit_cast(float, hi);
  }
}
__device__ __forceinline__ void unpack(const _Float16*, const u32x4& v, float (&f)[8]) {
  typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
  const f16x8 h = __builtin_bit_cast(f16x8, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
}
template <typename T, int VE>
__device__ __forceinline__ u32x4 pack(const float (&f)[VE]) {
  typedef __attribute__((ext_vector_type(VE))) T vec;
  vec v;
#pragma unroll
  for (int i = 0; i < VE; ++i) v[i] = (T)f[i];     // one rounding to nearest even, as a store of the product would do
  return __builtin_bit_cast(u32x4, v);
}

// span and element range [lo, hi) of a chunk; chunk < batch.chunks
struct ClipRange {
  int k;
  long lo, hi;
};
__device__ __forceinline__ ClipRange find_chunk(const ClipBatch& b, int chunk) {
  int a = 0, z = b.count - 1;
  while (a < z) {                    // first span whose chunk_end is beyond the chunk (uniform: scalar loads)
    const int m = (a + z) >> 1;
    if (b.chunk_end[m] > chunk) z = m;
    else a = m + 1;
  }
  const int first = a ? b.chunk_end[a - 1] : 0;
  const long per = b.chunk_bytes / (b.s[a].dtype == 0 ? 4 : 2);
  const long lo = (long)(chunk - first) * per;
  const long n = b.s[a].n;
  return {a, lo, lo + per < n ? lo + per : n};
}

// element index -> element offset of a span with rows of `cols` elements, `pitch` apart (cols == 0: contiguous)
__device__ __forceinline__ long span_at(long e, int cols, long pitch) {
  if (cols == 0) return e;
  const long r = (e >> 32) ? e / cols : (long)((unsigned)e / (unsigned)cols);
  return r * pitch + (e - r * cols);
}

template <typename T>
__device__ __forceinline__ double chunk_sumsq(const DtfClipSpan& s, long lo, long hi) {
  constexpr int VE = 16 / sizeof(T);
  const T* p = (const T*)s.in;
  double a0 = 0.0, a1 = 0.0, a2 = 0.0, a3 = 0.0;
  long v = lo / VE + threadIdx.x;                     // lo is a multiple of VE
  const bool whole = s.cols == 0 || s.cols % VE == 0; // no vector of elements crosses a row
  const long vend = whole ? hi / VE : 0;
  auto add = [&](const u32x4& x) {
    float f[VE];
    unpack(p, x, f);
#pragma unroll
    for (int i = 0; i < VE; i += 4) {
      a0 = fma((double)f[i], (double)f[i], a0);
      a1 = fma((double)f[i + 1], (double)f[i + 1], a1);
      a2 = fma((double)f[i + 2], (double)f[i + 2], a2);
      a3 = fma((double)f[i + 3], (double)f[i + 3], a3);
    }
  };
  if (s.cols == 0) {
    for (; v + 3 * kClipThreads < vend; v += 4 * kClipThreads) {   // four loads in flight
      u32x4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = load_any(p + (v + u * kClipThreads) * VE);
#pragma unroll
      for (int u = 0; u < 4; ++u) add(x[u]);
    }
  }
  for (; v < vend; v += kClipThreads) add(load_any(p + span_at(v * VE, s.cols, s.in_pitch)));
  for (long e = (whole ? (hi / VE) * VE : lo) + threadIdx.x; e < hi; e += kClipThreads) {
    const double f = (double)(float)p[span_at(e, s.cols, s.in_pitch)];
    a0 = fma(f, f, a0);
  }
  return (a0 + a1) + (a2 + a3);
}

// sum over the workgroup in a fixed order, the result in every thread
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(kClipThreads) void norm_partials(ClipBatch b, double* __restrict__ part) {
  __shared__ double red[4];
  double acc = 0.0;
  for (int c = blockIdx.x; c < b.chunks; c += gridDim.x) {
    const ClipRange r = find_chunk(b, c);
    const DtfClipSpan& s = b.s[r.k];
    acc += s.dtype == 0 ? chunk_sumsq<float>(s, r.lo, r.hi)
                        : s.dtype == 1 ? chunk_sumsq<bf16>(s, r.lo, r.hi) : chunk_sumsq<_Float16>(s, r.lo, r.hi);
  }
  acc = block_sum(acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// scale * sqrt(sum of the partial sums), the same bits in every thread of every workgroup
__device__ __forceinline__ double norm_of(const double* part, int np, double scale, double* red) {
  double a = 0.0;
  for (int i = threadIdx.x; i < np; i += kClipThreads) a += part[i];
  return scale * sqrt(block_sum(a, red));
}
// what a gradient value is multiplied with
__device__ __forceinline__ float clip_factor(double norm, double scale, double limit) {
  if (!(norm <= 1.7976931348623157e308)) return __builtin_nanf("");     // inf or NaN: every result says so
  return (float)(norm > limit ? scale * (limit / norm) : scale);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const DtfClipSpan& s, long lo, long hi, float f) {
  constexpr int VE = 16 / sizeof(T);
  const T* p = (const T*)s.in;
  T* o = (T*)s.out;
  const bool whole = s.cols == 0 || s.cols % VE == 0;
  const long vend = whole ? hi / VE : 0;
  long v = lo / VE + threadIdx.x;
  auto scaled = [&](const u32x4& x) {
    float y[VE];
    unpack(p, x, y);
#pragma unroll
    for (int i = 0; i < VE; ++i) y[i] *= f;
    return pack<T, VE>(y);
  };
  if (s.cols == 0) {
    for (; v + 3 * kClipThreads < vend; v += 4 * kClipThreads) {
      u32x4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = load_any(p + (v + u * kClipThreads) * VE);
#pragma unroll
      for (int u = 0; u < 4; ++u) store_any(o + (v + u * kClipThreads) * VE, scaled(x[u]));
    }
  }
  for (; v < vend; v += kClipThreads)
    store_any(o + span_at(v * VE, s.cols, s.out_pitch), scaled(load_any(p + span_at(v * VE, s.cols, s.in_pitch))));
  for (long e = (whole ? (hi / VE) * VE : lo) + threadIdx.x; e < hi; e += kClipThreads)
    o[span_at(e, s.cols, s.out_pitch)] = (T)((float)p[span_at(e, s.cols, s.in_pitch)] * f);
}

// in_place: the outputs are the inputs, and a factor of one leaves nothing to do
__global__ __launch_bounds__(kClipThreads) void clip_scale(ClipBatch b, const double* __restrict__ part, int np, double scale,
                                                           double limit, int in_place, float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double norm = norm_of(part, np, scale, red);
  const float f = clip_factor(norm, scale, limit);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  if (in_place && f == 1.0f) return;
  for (int c = b.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const ClipRange r = find_chunk(b, c);
    const DtfClipSpan& s = b.s[r.k];
    if (s.dtype == 0) chunk_scale<float>(s, r.lo, r.hi, f);
    else if (s.dtype == 1) chunk_scale<bf16>(s, r.lo, r.hi, f);
    else chunk_scale<_Float16>(s, r.lo, r.hi, f);
  }
}

// One workgroup: the norm alone, and -- hyper given -- the step's hyper-parameters with the gradient scale (hyper[4])
// multiplied by the factor, for update kernels that read them from device memory (optim.hip): the clipped update then
// needs no pass over the gradients.  The gradient scale itself is read from hyper, so a replayed graph follows it.
__global__ __launch_bounds__(kClipThreads) void norm_finish(const double* __restrict__ part, int np, double scale,
                                                            const float* __restrict__ hyper, float* __restrict__ hyper_out,
                                                            int n_hyper, double limit, float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double sc = hyper ? (double)hyper[4] : scale;
  const double norm = norm_of(part, np, sc, red);
  if (threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
  if (hyper && (int)threadIdx.x < n_hyper)
    hyper_out[threadIdx.x] = threadIdx.x == 4 ? clip_factor(norm, sc, limit) : hyper[threadIdx.x];
}

}  // namespace dtf

using namespace dtf;

static bool span_ok(const DtfClipSpan& s, bool need_out) {
  if (s.n < 0 || s.dtype < 0 || s.dtype > 2) return false;
  if (s.n == 0) return true;
  const uintptr_t align = s.dtype == 0 ? 3 : 1;
  if (!s.in || ((uintptr_t)s.in & align)) return false;
  if (need_out && (!s.out || ((uintptr_t)s.out & align))) return false;
  if (s.cols < 0 || (s.cols > 0 && (s.in_pitch < s.cols || (need_out && s.out_pitch < s.cols)))) return false;
  return true;
}

// Chunk size for all launches of one call: small totals are cut finer so that they spread over the chip.
static int chunk_bytes_for(int count, const DtfClipSpan* sp) {
  long bytes = 0;
  for (int k = 0; k < count; ++k) bytes += sp[k].n * (sp[k].dtype == 0 ? 4 : 2);
  long c = bytes / 2048 / kClipVec;         // about 2048 workgroups' worth
  c = c < 1 ? 1 : (c > 16 ? 16 : c);
  return (int)c * kClipVec;
}

// Walks the spans in batches of kSpans with at least one value each: fn(batch, grid).
template <class F>
static int for_batches(int count, const DtfClipSpan* sp, F&& fn) {
  ClipBatch b;
  b.chunk_bytes = chunk_bytes_for(count, sp);
  b.count = 0;
  b.chunks = 0;
  auto flush = [&]() -> int {
    if (!b.count) return 0;
    const int rc = fn(b, b.chunks < 2048 ? b.chunks : 2048);
    b.count = b.chunks = 0;
    return rc;
  };
  for (int k = 0; k < count; ++k) {
    if (!sp[k].n) continue;
    const long per = b.chunk_bytes / (sp[k].dtype == 0 ? 4 : 2);
    const long need = (sp[k].n + per - 1) / per;
    if (need > 0x3fffffff) return -3;        // 64 TB in one tensor
    if (b.count == kSpans || b.chunks > 0x3fffffff) {
      const int rc = flush();
      if (rc) return rc;
    }
    b.s[b.count] = sp[k];
    b.chunks += (int)need;
    b.chunk_end[b.count++] = b.chunks;
  }
  return flush();
}

extern "C" {

// fp64 slots of the partial-sum workspace that a call on these spans needs (at least 1); < 0: bad argument
long dtf_clip_partials(int count, const DtfClipSpan* spans) {
  if (count < 0 || (count && !spans)) return -3;
  for (int k = 0; k < count; ++k)
    if (!span_ok(spans[k], false)) return -3;
  long slots = 0;
  const int rc = for_batches(count, spans, [&](const ClipBatch&, int grid) { slots += grid; return 0; });
  return rc ? rc : (slots ? slots : 1);
}

static int partial_sums(int count, const DtfClipSpan* spans, double* part, long slots, long* used, hipStream_t s) {
  *used = 0;
  return for_batches(count, spans, [&](const ClipBatch& b, int grid) {
    if (*used + grid > slots) return -2;
    hipLaunchKernelGGL(norm_partials, dim3(grid), dim3(kClipThreads), 0, s, b, part + *used);
    *used += grid;
    return (int)hipGetLastError();
  });
}

// norm_out (fp32) = scale * norm of all spans.  With hyper / hyper_out (n_hyper floats, hyper[4] = the gradient scale, in
// place of `scale`) also hyper_out = hyper with [4] multiplied by limit / max(norm, limit); norm_out may then be NULL.
int dtf_global_norm(int count, const DtfClipSpan* spans, void* partials, long slots, double scale, const void* hyper,
                    void* hyper_out, int n_hyper, double limit, void* norm_out, hipStream_t s) {
  if (count < 0 || (count && !spans) || !partials || ((uintptr_t)partials & 7) || slots < 1) return -3;
  if (hyper ? (!hyper_out || n_hyper < 5 || n_hyper > kClipThreads || !(limit > 0.0)) : !norm_out) return -3;
  for (int k = 0; k < count; ++k)
    if (!span_ok(spans[k], false)) return -3;
  long used = 0;
  const int rc = partial_sums(count, spans, (double*)partials, slots, &used, s);
  if (rc) return rc;
  hipLaunchKernelGGL(norm_finish, dim3(1), dim3(kClipThreads), 0, s, (const double*)partials, (int)used, scale,
                     (const float*)hyper, (float*)hyper_out, n_hyper, limit, (float*)norm_out);
  return (int)hipGetLastError();
}

// out = in * scale * limit / max(norm, limit) for every span (out may be in itself), norm_out (fp32) = norm = scale * |in|
int dtf_clip_by_global_norm(int count, const DtfClipSpan* spans, void* partials, long slots, double scale, double limit,
                            void* norm_out, hipStream_t s) {
  if (count < 0 || (count && !spans) || !partials || ((uintptr_t)partials & 7) || slots < 1 || !norm_out) return -3;
  if (!(limit > 0.0) || !(limit <= 1.7976931348623157e308)) return -3;
  int in_place = 1;
  for (int k = 0; k < count; ++k) {
    if (!span_ok(spans[k], true)) return -3;
    if (spans[k].n && (spans[k].in != spans[k].out || (spans[k].cols && spans[k].in_pitch != spans[k].out_pitch))) in_place = 0;
  }
  long used = 0;
  int rc = partial_sums(count, spans, (double*)partials, slots, &used, s);
  if (rc) return rc;
  bool first = true;
  rc = for_batches(count, spans, [&](const ClipBatch& b, int grid) {
    hipLaunchKernelGGL(clip_scale, dim3(grid), dim3(kClipThreads), 0, s, b, (const double*)partials, (int)used, scale, limit,
                       in_place, first ? (float*)norm_out : nullptr);
    first = false;
    return (int)hipGetLastError();
  });
  if (rc || !first) return rc;
  // no values at all: the norm of nothing is zero
  hipLaunchKernelGGL(norm_finish, dim3(1), dim3(kClipThreads), 0, s, (const double*)partials, 0, scale, (const float*)nullptr,
                     (float*)nullptr, 0, 0.0, (float*)norm_out);
  return (int)hipGetLastError();
}

}  // extern "C"
