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
// the chunks in the opposite order and the last 192 MB of the first pass are the only ones it loads to stay, so that they are
// found in the 256 MB memory-side cache; everything else passes by it (non-temporal).  Measured, rotating over three lists:
// 0.72 G bf16 values 805 us with plain accesses, 785 with non-temporal stores, 719 with this (1.44 GB read twice and written
// once: 6.0 TB/s; a copy of that size runs at 5.0); 119 MB of mixed tensors 80 -> 61 us; norm of 209 MB 41.5 -> 36.7 us.
#include "common.hpp"
#include "api.h"

namespace dtf {

constexpr int kClipThreads = 256;
constexpr int kClipVec = kClipThreads * 16;   // bytes one workgroup reads per load instruction

// One chunk of one tensor, built on the host once per list (dtf_clip_table) and kept in device memory: a workgroup finds its
// work with a single 64-byte load, and a call over any number of tensors is two launches.  (The list as kernel arguments, 72
// tensors to a launch: 400 small tensors took 57 us, all of it launches.)
struct ClipChunk {
  const void* in;             // contiguous: of the chunk's first element; rows: of the tensor
  void* out;
  long lo;                    // rows: the chunk's first element
  long in_pitch, out_pitch;   // rows: elements between two of them
  int n;                      // elements
  int cols;                   // elements of a row; 0: contiguous
  int dtype;
  int pad[3];
};
static_assert(sizeof(ClipChunk) == 64, "one scalar load");

// 16 bytes at any element alignment (global memory takes unaligned vector accesses; a tensor of an arena may start at
// any element)
typedef u32x4 u32x4_any __attribute__((aligned(2)));
__device__ __forceinline__ u32x4 load_any(const void* p) {
  const u32x4 v = *reinterpret_cast<const u32x4_any*>(p);
  return v;
}
// the same, not to be kept in the caches
__device__ __forceinline__ u32x4 load_any_once(const void* p) {
  const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
  return v;
}
__device__ __forceinline__ void store_any_once(void* p, u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p)); }
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

// element index -> element offset of a tensor with rows of `cols` elements, `pitch` apart (cols == 0: contiguous)
__device__ __forceinline__ long span_at(long e, int cols, long pitch) {
  if (cols == 0) return e;
  const long r = (e >> 32) ? e / cols : (long)((unsigned)e / (unsigned)cols);
  return r * pitch + (e - r * cols);
}

// Walks the 16-byte vectors of a contiguous chunk, kDeep of them in flight per thread, then its last elements.  (Two to eight
// are within 2 % for large lists; four is best for those of 10 to 100 MB, where eight leave chunks to the one-vector loop.)
constexpr int kDeep = 4;
constexpr int kKeepChunks = 192 << 4;     // of 64 KB: 192 MB (smaller chunks belong to lists that fit the cache altogether)
template <typename T, bool PASS_BY>
__device__ __forceinline__ double chunk_sumsq(const ClipChunk& s) {
  constexpr int VE = 16 / sizeof(T);
  const T* p = (const T*)s.in;
  double a0 = 0.0, a1 = 0.0, a2 = 0.0, a3 = 0.0;
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
  auto one = [&](float x) { a0 = fma((double)x, (double)x, a0); };
  if (s.cols == 0) {
    const int vend = s.n / VE;
    int v = threadIdx.x;
    for (; v + (kDeep - 1) * kClipThreads < vend; v += kDeep * kClipThreads) {
      u32x4 x[kDeep];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const T* q = p + (v + u * kClipThreads) * VE;
        x[u] = PASS_BY ? load_any_once(q) : load_any(q);
      }
#pragma unroll
      for (int u = 0; u < kDeep; ++u) add(x[u]);
    }
    for (; v < vend; v += kClipThreads) add(load_any(p + v * VE));
    for (int e = vend * VE + threadIdx.x; e < s.n; e += kClipThreads) one((float)p[e]);
  } else if (s.cols % VE == 0) {       // no vector crosses a row (lo is a multiple of VE)
    for (int e = threadIdx.x * VE; e + VE <= s.n; e += kClipThreads * VE) add(load_any(p + span_at(s.lo + e, s.cols, s.in_pitch)));
  } else {
    for (int e = threadIdx.x; e < s.n; e += kClipThreads) one((float)p[span_at(s.lo + e, s.cols, s.in_pitch)]);
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

__global__ __launch_bounds__(kClipThreads) void norm_partials(const ClipChunk* __restrict__ table, int chunks, int keep,
                                                              double* __restrict__ part) {
  __shared__ double red[4];
  double acc = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const ClipChunk s = table[c];
    if (c < chunks - keep)
      acc += s.dtype == 0 ? chunk_sumsq<float, true>(s) : s.dtype == 1 ? chunk_sumsq<bf16, true>(s) : chunk_sumsq<_Float16, true>(s);
    else
      acc += s.dtype == 0 ? chunk_sumsq<float, false>(s) : s.dtype == 1 ? chunk_sumsq<bf16, false>(s) : chunk_sumsq<_Float16, false>(s);
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
// What a gradient value is multiplied with.  By the norm in 64 bits: that it is returned as infinity where fp32 does not hold it
// (two values of 3e38) makes no value wrong.
__device__ __forceinline__ double clip_factor(double norm, double scale, double limit) {
  if (!(norm <= 1.7976931348623157e308)) return __builtin_nan("");      // inf or NaN: every result says so
  return norm > limit ? scale * (limit / norm) : scale;
}
// The factor as m * 2^e: e is 0, but where it is subnormal in fp32 (limit 1e-3, norm 1e38: two digits left) or beyond it, and its
// products need not be.  m is then chosen so that x * m neither overflows (m <= 1 for small factors) nor loses digits of a small x
// (m from 2^126 on for large ones).
struct ClipFactor {
  float m;
  int e;
  __device__ __forceinline__ explicit ClipFactor(double c) : m((float)c), e(0) {
    if (!(c > 0.0)) return;
    if (m < 1.17549435e-38f) {
      m = (float)__builtin_amdgcn_frexp_mant(c);
      e = __builtin_amdgcn_frexp_exp(c);
    } else if (m > 3.40282347e38f) {
      m = (float)(__builtin_amdgcn_frexp_mant(c) * 0x1p127);
      e = __builtin_amdgcn_frexp_exp(c) - 127;
    }
  }
  __device__ __forceinline__ float times(float x) const { return __builtin_amdgcn_ldexpf(x * m, e); }
};

template <typename T>
__device__ __forceinline__ void chunk_scale(const ClipChunk& s, const ClipFactor& f) {
  constexpr int VE = 16 / sizeof(T);
  const T* p = (const T*)s.in;
  T* o = (T*)s.out;
  auto scaled = [&](const u32x4& x) {
    float y[VE];
    unpack(p, x, y);
#pragma unroll
    for (int i = 0; i < VE; ++i) y[i] = f.times(y[i]);
    return pack<T, VE>(y);
  };
  if (s.cols == 0) {
    const int vend = s.n / VE;
    int v = threadIdx.x;
    for (; v + (kDeep - 1) * kClipThreads < vend; v += kDeep * kClipThreads) {
      u32x4 x[kDeep];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) x[u] = load_any_once(p + (v + u * kClipThreads) * VE);
#pragma unroll
      for (int u = 0; u < kDeep; ++u) store_any_once(o + (v + u * kClipThreads) * VE, scaled(x[u]));
    }
    for (; v < vend; v += kClipThreads) store_any(o + v * VE, scaled(load_any(p + v * VE)));
    for (int e = vend * VE + threadIdx.x; e < s.n; e += kClipThreads) o[e] = (T)f.times((float)p[e]);
  } else if (s.cols % VE == 0) {
    for (int e = threadIdx.x * VE; e + VE <= s.n; e += kClipThreads * VE)
      store_any(o + span_at(s.lo + e, s.cols, s.out_pitch), scaled(load_any(p + span_at(s.lo + e, s.cols, s.in_pitch))));
  } else {
    for (int e = threadIdx.x; e < s.n; e += kClipThreads)
      o[span_at(s.lo + e, s.cols, s.out_pitch)] = (T)f.times((float)p[span_at(s.lo + e, s.cols, s.in_pitch)]);
  }
}

// in_place: the outputs are the inputs, and a factor of one leaves nothing to do
__global__ __launch_bounds__(kClipThreads) void clip_scale(const ClipChunk* __restrict__ table, int chunks,
                                                           const double* __restrict__ part, int np, double scale, double limit,
                                                           int in_place, float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double norm = norm_of(part, np, scale, red);
  const ClipFactor f(clip_factor(norm, scale, limit));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  if (in_place && f.m == 1.0f && f.e == 0) return;
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const ClipChunk s = table[c];
    if (s.dtype == 0) chunk_scale<float>(s, f);
    else if (s.dtype == 1) chunk_scale<bf16>(s, f);
    else chunk_scale<_Float16>(s, f);
  }
}

// One workgroup: the norm alone, and -- hyper given -- the step's hyper-parameters with the gradient scale (hyper[4])
// multiplied by the factor, for update kernels that read them from device memory (optim.hip): the clipped update then
// needs no pass over the gradients.  The gradient scale itself is read from hyper, so a replayed graph follows it.  (The factor is
// an fp32 number like the others there: below 1.2e-38, a norm of 1e38 against a limit of 1, it loses digits.)
__global__ __launch_bounds__(kClipThreads) void norm_finish(const double* __restrict__ part, int np, double scale,
                                                            const float* __restrict__ hyper, float* __restrict__ hyper_out,
                                                            int n_hyper, double limit, float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double sc = hyper ? (double)hyper[4] : scale;
  const double norm = norm_of(part, np, sc, red);
  if (threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
  if (hyper && (int)threadIdx.x < n_hyper)
    hyper_out[threadIdx.x] = threadIdx.x == 4 ? (float)clip_factor(norm, sc, limit) : hyper[threadIdx.x];
}

}  // namespace dtf

using namespace dtf;

static int clip_grid(long chunks) { return (int)(chunks < 2048 ? (chunks < 1 ? 1 : chunks) : 2048); }

extern "C" {

// Number of chunks of a list of tensors (< 0: bad argument).  table != NULL: 64 bytes per chunk are written there (host memory),
// to be copied to the device; *in_place = whether every output is its input.
long dtf_clip_table(int count, const DtfClipSpan* spans, void* table, long table_chunks, int* in_place) {
  if (count < 0 || (count && !spans)) return -3;
  long bytes = 0;
  int same = 1;
  for (int k = 0; k < count; ++k) {
    const DtfClipSpan& s = spans[k];
    if (s.n < 0 || s.dtype < 0 || s.dtype > 2) return -3;
    if (s.n == 0) continue;
    const int E = s.dtype == 0 ? 4 : 2;
    if (!s.in || ((uintptr_t)s.in & (E - 1)) || !s.out || ((uintptr_t)s.out & (E - 1))) return -3;
    if (s.cols < 0 || (s.cols > 0 && (s.in_pitch < s.cols || s.out_pitch < s.cols || s.n % s.cols))) return -3;
    if (s.in != s.out || (s.cols && s.in_pitch != s.out_pitch)) same = 0;
    bytes += s.n * E;
  }
  if (in_place) *in_place = same;
  // About 2048 chunks, one workgroup each; small lists are cut into 4 KB, large ones into 64 KB.
  long per = bytes / 2048 / kClipVec;
  per = (per < 1 ? 1 : (per > 16 ? 16 : per)) * kClipVec;
  long chunks = 0;
  ClipChunk* t = (ClipChunk*)table;
  for (int k = 0; k < count; ++k) {
    const DtfClipSpan& s = spans[k];
    const int E = s.dtype == 0 ? 4 : 2;
    const long step = per / E;
    for (long lo = 0; lo < s.n; lo += step, ++chunks) {
      if (chunks >= 0x7fffffff) return -1;
      if (!t) continue;
      if (chunks >= table_chunks) return -2;
      const int n = (int)(s.n - lo < step ? s.n - lo : step);
      const long at = s.cols ? 0 : lo * E;
      t[chunks] = ClipChunk{(const char*)s.in + at, (char*)s.out + at, s.cols ? lo : 0, s.in_pitch, s.out_pitch, n, s.cols, s.dtype, {0, 0, 0}};
    }
  }
  return chunks;
}

// fp64 words of a call's workspace
long dtf_clip_partials(long chunks) { return chunks < 0 ? -3 : clip_grid(chunks); }

static bool table_ok(const void* table, long chunks, const void* partials, long slots) {
  return chunks >= 0 && chunks <= 0x7fffffff && (table || !chunks) && !((uintptr_t)table & 63) && partials && !((uintptr_t)partials & 7) &&
         slots >= clip_grid(chunks);
}

// norm_out (fp32) = scale * norm of the table's tensors.  With hyper / hyper_out (n_hyper floats, hyper[4] = the gradient scale,
// in place of `scale`) also hyper_out = hyper with [4] multiplied by limit / max(norm, limit); norm_out may then be NULL.
int dtf_global_norm(const void* table, long chunks, void* partials, long slots, double scale, const void* hyper, void* hyper_out,
                    int n_hyper, double limit, void* norm_out, hipStream_t s) {
  if (!table_ok(table, chunks, partials, slots)) return -3;
  if (hyper ? (!hyper_out || n_hyper < 5 || n_hyper > kClipThreads || !(limit > 0.0)) : !norm_out) return -3;
  const int grid = clip_grid(chunks);
  hipLaunchKernelGGL(norm_partials, dim3(grid), dim3(kClipThreads), 0, s, (const ClipChunk*)table, (int)chunks,
                     hyper ? kKeepChunks : 0, (double*)partials);      // (an update reads the gradients next, a bare norm nothing)
  hipLaunchKernelGGL(norm_finish, dim3(1), dim3(kClipThreads), 0, s, (const double*)partials, grid, scale, (const float*)hyper,
                     (float*)hyper_out, n_hyper, limit, (float*)norm_out);
  return (int)hipGetLastError();
}

// out = in * scale * limit / max(norm, limit) for every tensor of the table, norm_out (fp32) = norm = scale * |in|
int dtf_clip_by_global_norm(const void* table, long chunks, int in_place, void* partials, long slots, double scale, double limit,
                            void* norm_out, hipStream_t s) {
  if (!table_ok(table, chunks, partials, slots) || !norm_out || !(limit > 0.0) || !(limit <= 1.7976931348623157e308)) return -3;
  const int grid = clip_grid(chunks);
  hipLaunchKernelGGL(norm_partials, dim3(grid), dim3(kClipThreads), 0, s, (const ClipChunk*)table, (int)chunks, kKeepChunks,
                     (double*)partials);
  hipLaunchKernelGGL(clip_scale, dim3(grid), dim3(kClipThreads), 0, s, (const ClipChunk*)table, (int)chunks, (const double*)partials, grid,
                     scale, limit, in_place, (float*)norm_out);
  return (int)hipGetLastError();
}

}  // extern "C"
