// Classifier head with many classes: softmax cross-entropy over the product of the hidden rows with a [classes][hidden]
// weight, forward and backward, without ever storing the logits (head.hip is the ten-class form, whose logits fit in
// registers):
//   z_iv = h_i . w_v + b_v      lse_i = log sum_v exp(z_iv)      loss_i = lse_i - z_iy
//   d_iv = s_i (exp(z_iv - lse_i) - [v = y_i])      dh = d . w      dw = d^T . h      db_v = sum_i d_iv
// Forward: one pass of the logits product; a tile's logits live in its accumulators, the epilogue reduces them to one
// (maximum, sum of exponentials) pair per row and class tile, and a small kernel joins the pairs.
// Backward: for one piece of the classes after the other the logits are computed again (8 n H V operations in all
// instead of the 6 n H V of a program that keeps n V logits), d of that piece is stored in the operand type, and two more
// products make dw of the piece and add to dh, which is summed over the pieces in fp32.
//
// All products run through one kernel, vh_gemm: out[j][i] = sum_k A[i][k] B[j][k], both operands with contiguous k.
#include "common.hpp"
#include "api.h"

namespace dtf {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
typedef f32x4 f32x4_any __attribute__((aligned(4)));

template <typename T> struct VhType;
template <> struct VhType<bf16> {
  static constexpr int KE = 32;     // elements of a 64-byte K tile row
  typedef bf16x8 Vec;               // 16 bytes
  static __device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, f32x4 c) {
    return mfma16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
  }
};
template <> struct VhType<float> {
  static constexpr int KE = 16;
  typedef f32x4 Vec;
  // lane group g holds k = 4 g .. 4 g + 3 of both operands; step s multiplies k = 4 g + s, so that the four steps cover
  // all sixteen
  static __device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, f32x4 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s], y[s], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ void vh_dma16(__amdgpu_buffer_rsrc_t r, const void* lds, uint32_t voff, uint32_t soff) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) void lds_void;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, voff, soff, 0, 0);
#else
  (void)r; (void)lds; (void)voff; (void)soff;
#endif
}

// Wait until at most VM of this wave's LDS-DMAs are in flight and all its LDS reads have returned.  The builtin (not asm),
// so that the compiler knows it too and adds no waits of its own; nothing that touches memory moves across.
template <int VM>
__device__ __forceinline__ void vh_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((VM & 15) | 0x70 | ((VM >> 4) << 14));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void vh_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct VhTrue { static constexpr bool value = true; };
struct VhFalse { static constexpr bool value = false; };

struct VhOperands {
  const void *A, *B;      // rows of K elements, lda / ldb elements apart, 16-byte aligned
  long lda, ldb;
  int M, N, K;            // K: a multiple of 16 bytes
  int tiles_m, tiles_n;
};

// C tile of a wave: lane l holds rows i = 16 mt + 4 (l >> 4) + r, column j = 16 nt + (l & 15) -- four consecutive i
// (classes, or hidden units) of one j.
template <typename T, int BM, int BN, int NWM, int NWN>
struct VhTile {
  static constexpr int NT = NWM * NWN * 64;
  static constexpr int WM = BM / NWM, WN = BN / NWN, MT = WM / 16, NTL = WN / 16;
  f32x4 acc[MT][NTL];
  int m0, n0;             // of the workgroup's tile
  int wm0, wn0;           // of the wave's tile, within the workgroup's
  int lane, wave;
};

// Main loop.  K tiles of 64 bytes per row, D buffers in LDS, filled by LDS-DMA; rows of 64 bytes, the 16-byte chunk p of row
// r holds chunk p ^ ((r >> 1) & 3), so that the fragment reads of 16 rows touch every bank once.
// Phase t: DMA of tile t + D into the buffer of tile t (whose fragments every wave read before the last barrier) | read the
// fragments of tile t + 1 | MFMAs on those of tile t | wait until tile t + 2 has landed | barrier.
template <typename T, int BM, int BN, int NWM, int NWN, int D, class Tile>
__device__ __forceinline__ void vh_mainloop(const VhOperands& p, Tile& c, char* lds) {
  constexpr int NT = Tile::NT, MT = Tile::MT, NTL = Tile::NTL;
  constexpr int ACH = BM * 4 / NT, BCH = BN * 4 / NT, NDMA = ACH + BCH;
  static_assert(BM * 4 % NT == 0 && BN * 4 % NT == 0, "every thread stages whole chunks");
  constexpr int ABYTES = BM * 64, STAGE = (BM + BN) * 64;
  const int tid = threadIdx.x, lane = c.lane, i16 = lane & 15, g = lane >> 4;
  const int E = (int)sizeof(T);
  const int rows_a = min(BM, p.M - c.m0), rows_b = min(BN, p.N - c.n0);
  const __amdgpu_buffer_rsrc_t ra = make_rsrc((const char*)p.A + (size_t)c.m0 * p.lda * E, ((size_t)(rows_a - 1) * p.lda + p.K) * E);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc((const char*)p.B + (size_t)c.n0 * p.ldb * E, ((size_t)(rows_b - 1) * p.ldb + p.K) * E);
  uint32_t va[ACH], vb[BCH];
#pragma unroll
  for (int i = 0; i < ACH; ++i) {
    const int q = tid + i * NT, row = q >> 2;
    va[i] = (uint32_t)row * (uint32_t)(p.lda * E) + (((q & 3) ^ ((row >> 1) & 3)) << 4);
  }
#pragma unroll
  for (int i = 0; i < BCH; ++i) {
    const int q = tid + i * NT, row = q >> 2;
    vb[i] = (uint32_t)row * (uint32_t)(p.ldb * E) + (((q & 3) ^ ((row >> 1) & 3)) << 4);
  }
  const int kbytes = p.K * E, T_ = (kbytes + 63) >> 6;
  // chunks of a lane: byte offset of its chunk within the 64-byte row (the same for every i: NT is a multiple of 8 rows)
  const int kch = (((tid & 3) ^ ((tid >> 3) & 3)) << 4);
  auto dma = [&](int t, int buf) {
    const uint32_t so = (uint32_t)t << 6;
    const bool in = (int)so + kch < kbytes;          // the last K tile may end inside the row: zeros from there on
    char* const base = lds + buf * STAGE + c.wave * 1024;
#pragma unroll
    for (int i = 0; i < ACH; ++i) vh_dma16(ra, base + i * NT * 16, in ? va[i] : 0xfffffff0u, so);
#pragma unroll
    for (int i = 0; i < BCH; ++i) vh_dma16(rb, base + ABYTES + i * NT * 16, in ? vb[i] : 0xfffffff0u, so);
  };
  u32x4 fa[2][MT], fb[2][NTL];
  const int sw = (g ^ ((i16 >> 1) & 3)) << 4;
  const int oa = (c.wm0 + i16) * 64 + sw, ob = ABYTES + (c.wn0 + i16) * 64 + sw;
  auto frags = [&](u32x4 (&a)[MT], u32x4 (&b)[NTL], int buf) {
    const char* base = lds + buf * STAGE;
#pragma unroll
    for (int i = 0; i < MT; ++i) a[i] = *reinterpret_cast<const u32x4*>(base + oa + i * 1024);
#pragma unroll
    for (int j = 0; j < NTL; ++j) b[j] = *reinterpret_cast<const u32x4*>(base + ob + j * 1024);
  };
  auto mma = [&](const u32x4 (&a)[MT], const u32x4 (&b)[NTL]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NTL; ++j) c.acc[i][j] = VhType<T>::mma(a[i], b[j], c.acc[i][j]);
  };
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NTL; ++j) c.acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < T_) dma(d, d);
  if (T_ >= D) vh_wait<(D - 2) * NDMA>();
  else vh_wait<0>();
  vh_barrier();
  frags(fa[0], fb[0], 0);
  vh_wait<63>();
  vh_barrier();
  int buf = 0;
  // steady: tiles t + 1 and t + D exist
  auto phase = [&](auto steady, int t, u32x4 (&a)[MT], u32x4 (&b)[NTL], u32x4 (&na)[MT], u32x4 (&nb)[NTL]) {
    constexpr bool kSteady = decltype(steady)::value;
    const bool more = kSteady || t + D < T_;
    if (more) dma(t + D, buf);
    buf = buf + 1 == D ? 0 : buf + 1;
    if (kSteady || t + 1 < T_) frags(na, nb, buf);
    mma(a, b);
    if (kSteady) {
      vh_wait<(D - 2) * NDMA>();
    } else {
      vh_wait<63>();                      // the LDS reads, on every path
      if (!more) vh_wait<0>();
      else vh_wait<(D - 2) * NDMA>();
    }
    vh_barrier();
  };
  int t = 0;
#pragma unroll 1
  for (; t + 1 + D < T_; t += 2) {
    phase(VhTrue{}, t, fa[0], fb[0], fa[1], fb[1]);
    phase(VhTrue{}, t + 1, fa[1], fb[1], fa[0], fb[0]);
  }
#pragma unroll 1
  for (; t < T_; t += 2) {
    phase(VhFalse{}, t, fa[0], fb[0], fa[1], fb[1]);
    if (t + 1 < T_) phase(VhFalse{}, t + 1, fa[1], fb[1], fa[0], fb[0]);
  }
}

template <typename T, int BM, int BN, int NWM, int NWN, int D, class Epi>
__global__ __launch_bounds__(NWM * NWN * 64, 1) void vh_gemm(VhOperands p, Epi e) {
  typedef VhTile<T, BM, BN, NWM, NWN> Tile;
  __shared__ __attribute__((aligned(16))) char lds[D * (BM + BN) * 64];
  Tile c;
  c.lane = threadIdx.x & 63;
  c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  c.wm0 = (c.wave / NWN) * Tile::WM;
  c.wn0 = (c.wave % NWN) * Tile::WN;
  int tx, ty;
  xcd_tile_linear(blockIdx.x, p.tiles_m, p.tiles_n, tx, ty);
  c.m0 = tx * BM;
  c.n0 = ty * BN;
  vh_mainloop<T, BM, BN, NWM, NWN, D>(p, c, lds);
  e.template run<T, BM, BN, NWM, NWN>(p, c, tx, ty, lds);
}

// ---- epilogues ------------------------------------------------------------------------------------------------------
// Logits of a lane's four consecutive classes: bias added, classes beyond the last one -inf.
__device__ __forceinline__ f32x4 vh_bias4(const float* bias, int m, int M) {
  f32x4 b = {0.f, 0.f, 0.f, 0.f};
  if (bias) {
    if (m + 4 <= M) b = *reinterpret_cast<const f32x4_any*>(bias + m);
    else
#pragma unroll
      for (int r = 0; r < 4; ++r) b[r] = m + r < M ? bias[m + r] : 0.f;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) b[r] = m + r < M ? b[r] : -INFINITY;
  return b;
}

// (a.m, a.s) stands for a.s * exp2(a.m): the sum of exponentials relative to the largest.  An empty sum is (-inf, 0).
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s};          // (nothing to rescale; exp2(-inf + inf) would be NaN)
  return {m, a.s * exp2f(a.m - m) + b.s * exp2f(b.m - m)};
}

// Forward: i = class, j = row.  part[class tile][row] = (maximum, sum) in base 2, zlab[row] = the label's logit.
struct VhForward {
  const float* bias;
  const int* labels;
  float2* part;
  float* zlab;
  long ldpart;
  template <typename T, int BM, int BN, int NWM, int NWN, class Tile>
  __device__ void run(const VhOperands& p, Tile& c, int tx, int, char* lds) const {
    constexpr int MT = Tile::MT, NTL = Tile::NTL;
    const int i16 = c.lane & 15, g = c.lane >> 4;
    const int mw = c.m0 + c.wm0 + 4 * g;
    MaxSum (*red)[BN] = reinterpret_cast<MaxSum(*)[BN]>(lds);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const f32x4 b = vh_bias4(bias, mw + 16 * i, p.M);
#pragma unroll
      for (int j = 0; j < NTL; ++j) c.acc[i][j] += b;
    }
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
      const int row = c.n0 + c.wn0 + 16 * j + i16;
      const int y = row < p.N ? labels[row] - mw : -1;      // label relative to this lane's first class
      if (__any(y >= 0 && y < Tile::WM)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (y == 16 * i + r) zlab[row] = c.acc[i][j][r];
      }
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, c.acc[i][j][r]);
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float m2 = m * kLog2e, off = m == -INFINITY ? 0.f : m2;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f(fmaf(c.acc[i][j][r], kLog2e, -off));
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if (g == 0) red[c.wave / NWN][c.wn0 + 16 * j + i16] = {m2, s};
    }
    __syncthreads();
    for (int j = threadIdx.x; j < BN; j += Tile::NT) {
      MaxSum a = red[0][j];
#pragma unroll
      for (int w = 1; w < NWM; ++w) a = join(a, red[w][j]);
      if (c.n0 + j < p.N) part[(long)tx * ldpart + c.n0 + j] = make_float2(a.m, a.s);
    }
  }
};

// Backward, first product: i = class (relative to the piece), j = row.  d[row][class] in the operand type, columns up to
// ldd (a multiple of the K tile) written as zeros; dbias partial sums per row tile from the values before rounding.
struct VhGradLogits {
  const float* bias;        // of the piece
  const int* labels;
  const float* lse;
  const float* row_scale;   // or nullptr
  float grad_scale;
  int v0, classes, ignore;
  void* d;
  long ldd;
  float* dbpart;            // [row tile][ldd] or nullptr
  template <typename T, int BM, int BN, int NWM, int NWN, class Tile>
  __device__ void run(const VhOperands& p, Tile& c, int, int ty, char* lds) const {
    constexpr int MT = Tile::MT, NTL = Tile::NTL;
    const int i16 = c.lane & 15, g = c.lane >> 4;
    const int mw = c.m0 + c.wm0 + 4 * g;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const f32x4 b = vh_bias4(bias, mw + 16 * i, p.M);
#pragma unroll
      for (int j = 0; j < NTL; ++j) c.acc[i][j] += b;
    }
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
      const int row = c.n0 + c.wn0 + 16 * j + i16;
      const bool live = row < p.N;
      const int label = live ? labels[row] : ignore;
      float sc = label == ignore ? 0.f : (row_scale ? grad_scale * row_scale[row] : grad_scale);
      const float l2 = live ? lse[row] * kLog2e : 0.f;
      const bool known = label >= 0 && label < classes;
      if (label != ignore && !known) sc = __builtin_nanf("");       // a label that is no class: the whole row says so
      const int y = known ? label - v0 - mw : -1;
      const bool dead = label == ignore;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // (an ignored row is zero whatever its logits are)
          const float e = __builtin_amdgcn_exp2f(fmaf(c.acc[i][j][r], kLog2e, -l2));
          v[r] = dead ? 0.f : sc * (y == 16 * i + r ? e - 1.f : e);
        }
        c.acc[i][j] = v;
        const int m = mw + 16 * i;
        if (live && m < ldd) {
          typedef __attribute__((ext_vector_type(4))) T T4;
          const T4 o = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
          *reinterpret_cast<T4*>((T*)d + (long)row * ldd + m) = o;
        }
      }
    }
    if (!dbpart) return;
    float (*red)[BM] = reinterpret_cast<float(*)[BM]>(lds);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      f32x4 s = c.acc[i][0];
#pragma unroll
      for (int j = 1; j < NTL; ++j) s += c.acc[i][j];
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = row16_sum(s[r]);
      if (i16 == 0) *reinterpret_cast<f32x4*>(&red[c.wave % NWN][c.wm0 + 16 * i + 4 * g]) = s;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < BM; i += Tile::NT) {
      float s = red[0][i];
#pragma unroll
      for (int w = 1; w < NWN; ++w) s += red[w][i];
      if (c.m0 + i < ldd) dbpart[(long)ty * ldd + c.m0 + i] = s;
    }
  }
};

// Plain product: out[j][i] in type O; acc: fp32 [N][M] running sum over the pieces of the classes (read unless `first`,
// written unless `last`, in which case the result goes to out).
struct VhStore {
  void* out;
  long ldo;
  int out_f32;              // out holds fp32, else the operand type
  float* sum;               // nullptr: a single piece
  int first, last;
  template <typename T, int BM, int BN, int NWM, int NWN, class Tile>
  __device__ void run(const VhOperands& p, Tile& c, int, int, char*) const {
    constexpr int MT = Tile::MT, NTL = Tile::NTL;
    const int i16 = c.lane & 15, g = c.lane >> 4;
    const bool vec = !(p.M & 3);
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
      const int row = c.n0 + c.wn0 + 16 * j + i16;
      if (row >= p.N) continue;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = c.m0 + c.wm0 + 16 * i + 4 * g;
        if (m >= p.M) continue;
        f32x4 v = c.acc[i][j];
        const int left = p.M - m;
        float* s = sum ? sum + (long)row * p.M + m : nullptr;
        if (s && !first) {
          if (vec) v += *reinterpret_cast<const f32x4*>(s);
          else
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += r < left ? s[r] : 0.f;
        }
        if (s && !last) {
          if (vec) *reinterpret_cast<f32x4*>(s) = v;
          else
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r < left) s[r] = v[r];
          continue;
        }
        if (out_f32 || sizeof(T) == 4) {
          float* o = (float*)out + (long)row * ldo + m;
          if (vec) *reinterpret_cast<f32x4_any*>(o) = v;
          else
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r < left) o[r] = v[r];
        } else {
          T* o = (T*)out + (long)row * ldo + m;
          typedef __attribute__((ext_vector_type(4))) T T4;
          typedef T4 T4_any __attribute__((aligned(2)));
          const T4 x = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
          if (vec) *reinterpret_cast<T4_any*>(o) = x;
          else
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r < left) o[r] = x[r];
        }
      }
    }
  }
};

// ---- small kernels --------------------------------------------------------------------------------------------------
// lse and loss of a row from its (maximum, sum) pairs, joined in class order: 16 rows x 16 slices per workgroup.
__global__ __launch_bounds__(256) void vh_join(const float2* __restrict__ part, long ldpart, int tiles, const float* __restrict__ zlab,
                                               const int* __restrict__ labels, int n, int classes, int ignore,
                                               float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ MaxSum red[16][17];
  const int rl = threadIdx.x & 15, sl = threadIdx.x >> 4, row = blockIdx.x * 16 + rl;
  MaxSum a = {-INFINITY, 0.f};
  if (row < n) {
    const int per = (tiles + 15) / 16, t1 = min(tiles, (sl + 1) * per);
    for (int t = sl * per; t < t1; ++t) {
      const float2 v = part[(long)t * ldpart + row];
      a = join(a, {v.x, v.y});
    }
  }
  red[sl][rl] = a;
  __syncthreads();
  if (sl || row >= n) return;
  for (int w = 1; w < 16; ++w) a = join(a, red[w][rl]);
  const float l = kLn2 * (a.m + __builtin_amdgcn_logf(a.s));     // (the hardware's base-2 logarithm, one step of error)
  lse[row] = l;
  const int y = labels[row];
  loss[row] = y == ignore ? 0.f : (y >= 0 && y < classes ? l - zlab[row] : __builtin_nanf(""));
}

// db[v] = sum of the row tiles' partial sums, in order
__global__ __launch_bounds__(256) void vh_dbias(const float* __restrict__ part, long ld, int tiles, float* __restrict__ db, int n) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= n) return;
  float s = 0.f;
  for (int t = 0; t < tiles; ++t) s += part[(long)t * ld + v];
  db[v] = s;
}

// dst[c][r] = src[r][c] for r < R, c < C; columns R .. ldd - 1 of dst are zero.  Rows of src for which live(r) is false
// count as zero (labels given: the ignored ones -- whatever lies there, 0 * NaN must not reach a gradient).
// 64 x 64 tiles through LDS.
template <typename T>
__global__ __launch_bounds__(256) void vh_transpose(const T* __restrict__ src, long lds_, int R, int C, T* __restrict__ dst, long ldd,
                                                    const int* __restrict__ labels, int ignore) {
  __shared__ T tile[64][64 + 4 / sizeof(T) * 2];
  const int nr = (int)((ldd + 63) >> 6);
  const int r0 = (blockIdx.x % nr) * 64, c0 = (blockIdx.x / nr) * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (int i = y; i < 64; i += 4) {
    const int r = r0 + i, c = c0 + x;
    T v = (T)0.f;
    if (r < R && c < C && !(labels && labels[r] == ignore)) v = src[(long)r * lds_ + c];
    tile[i][x] = v;
  }
  __syncthreads();
  for (int i = y; i < 64; i += 4) {
    const int c = c0 + i, r = r0 + x;
    if (c < C && r < ldd) dst[(long)c * ldd + r] = tile[x][i];
  }
}

// dst[r][c] = src[r][c] with rows ldd apart, columns C .. ldd - 1 zero: a copy whose rows start on 16 bytes
template <typename T>
__global__ __launch_bounds__(256) void vh_pad(const T* __restrict__ src, long lds_, int R, int C, T* __restrict__ dst, long ldd) {
  const long n = (long)R * ldd;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / ldd;
    const int c = (int)(i - r * ldd);
    dst[i] = c < C ? src[r * lds_ + c] : (T)0.f;
  }
}

}  // namespace dtf

using namespace dtf;

namespace {

constexpr long up(long a, long b) { return (a + b - 1) / b * b; }
constexpr int cdiv(long a, long b) { return (int)((a + b - 1) / b); }
constexpr int kTile = 256;            // classes per tile of the logits products: the partials are laid out by it
constexpr long kMaxRow = 1L << 20;    // longest row of an operand: a tile's 256 rows are addressed with 32-bit byte offsets
template <typename T> constexpr int kRows = sizeof(T) == 2 ? 256 : 128;      // rows of h per tile

template <typename T, class Epi>
int run_gemm(VhOperands p, const Epi& e, hipStream_t s) {
  constexpr int BM = kTile, BN = kRows<T>;
  p.tiles_m = cdiv(p.M, BM);
  p.tiles_n = cdiv(p.N, BN);
  hipLaunchKernelGGL((vh_gemm<T, BM, BN, 2, sizeof(T) == 2 ? 4 : 2, 4, Epi>), dim3(p.tiles_m * p.tiles_n),
                     dim3(sizeof(T) == 2 ? 512 : 256), 0, s, p, e);
  return (int)hipGetLastError();
}

// Layout of one call's workspace (bytes).  Everything a call needs besides its inputs and outputs.
struct Plan {
  long h_pad, w_pad;        // 16-byte aligned copies of h / of a piece of w (0: used as they are)
  long part, zlab;          // forward
  long hT, wT, d, dT, sum, dbpart;
  long total;
  long ldk, ldn, ldv;       // padded hidden, rows, classes of a piece
  int piece, pieces, row_tiles;
};

int esize(int dtype) { return dtype == 1 ? 2 : 4; }

// Classes per piece: d and its transpose take piece * n values each.  2^27 values (256 MB in bf16) leave few, long pieces --
// every piece reads and writes the fp32 sum of dh once.
int piece_for(long n, int classes) {
  long v = (1L << 27) / (n < 1 ? 1 : n) / kTile * kTile;
  if (v < 4 * kTile) v = 4 * kTile;
  if (v > kMaxRow) v = kMaxRow;
  return v >= classes ? classes : (int)v;
}

Plan plan_for(int dtype, int backward, long n, int H, int V, bool h_ok, bool w_ok, bool bias, int piece) {
  Plan q{};
  const int E = esize(dtype), KE = 64 / E;
  long at = 0;
  auto take = [&](long bytes) {
    const long o = at;
    at += up(bytes, 256);
    return o + 1;           // 0 stands for "none"
  };
  q.ldk = up(H, 16 / E);
  q.ldn = up(n, KE);
  if (!h_ok) q.h_pad = take(n * q.ldk * E);
  q.piece = backward ? (piece > 0 ? (int)up(piece, kTile) : piece_for(n, V)) : V;
  if (q.piece > V) q.piece = V;
  q.pieces = cdiv(V, q.piece);
  if (!w_ok) q.w_pad = take((long)q.piece * q.ldk * E);
  if (!backward) {
    q.part = take((long)cdiv(V, kTile) * n * 8);
    q.zlab = take(n * 4);
  } else {
    q.ldv = up(q.piece, KE);
    q.row_tiles = cdiv(n, E == 2 ? kRows<bf16> : kRows<float>);
    q.hT = take(H * q.ldn * E);
    q.wT = take(H * q.ldv * E);
    q.d = take(n * q.ldv * E);
    q.dT = take(q.piece * q.ldn * E);
    if (q.pieces > 1) q.sum = take(n * H * 4);
    if (bias) q.dbpart = take((long)q.row_tiles * q.ldv * 4);
  }
  q.total = at ? at : 256;
  return q;
}

template <typename T>
T* at(void* ws, long o) { return (T*)((char*)ws + o - 1); }

bool rows_ok(const void* p, long ld, int H, int E) { return !((uintptr_t)p & 15) && !(ld * E & 15) && !((long)H * E & 15); }

template <typename T>
int launch_transpose(const T* src, long lds, int R, int C, T* dst, long ldd, const int* labels, int ignore, hipStream_t s) {
  hipLaunchKernelGGL(vh_transpose<T>, dim3(cdiv(C, 64) * cdiv(ldd, 64)), dim3(256), 0, s, src, lds, R, C, dst, ldd, labels, ignore);
  return (int)hipGetLastError();
}
template <typename T>
int launch_pad(const T* src, long lds, int R, int C, T* dst, long ldd, hipStream_t s) {
  const long blocks = cdiv((long)R * ldd, 1024);
  hipLaunchKernelGGL(vh_pad<T>, dim3(blocks > 8192 ? 8192 : (int)blocks), dim3(256), 0, s, src, lds, R, C, dst, ldd);
  return (int)hipGetLastError();
}

#define VH_TRY(x)             \
  do {                        \
    const int rc_ = (x);      \
    if (rc_ != 0) return rc_; \
  } while (0)

template <typename T>
int forward(const void* h, long ldh, const void* w, long ldw, const float* bias, const int* labels, int n, int H, int V, int ignore,
            void* loss, void* lse, void* ws, hipStream_t s) {
  const int E = sizeof(T);
  const bool h_ok = rows_ok(h, ldh, H, E), w_ok = rows_ok(w, ldw, H, E);
  const Plan q = plan_for(E == 2 ? 1 : 0, 0, n, H, V, h_ok, w_ok, bias != nullptr, 0);
  VhOperands p{w, h, ldw, ldh, V, n, H, 0, 0};
  if (!h_ok) {
    VH_TRY(launch_pad((const T*)h, ldh, n, H, at<T>(ws, q.h_pad), q.ldk, s));
    p.B = at<T>(ws, q.h_pad);
    p.ldb = q.ldk;
  }
  if (!w_ok) {
    VH_TRY(launch_pad((const T*)w, ldw, V, H, at<T>(ws, q.w_pad), q.ldk, s));
    p.A = at<T>(ws, q.w_pad);
    p.lda = q.ldk;
  }
  p.K = (int)q.ldk;
  VhForward e{bias, labels, at<float2>(ws, q.part), at<float>(ws, q.zlab), n};
  VH_TRY((run_gemm<T>(p, e, s)));
  hipLaunchKernelGGL(vh_join, dim3(cdiv(n, 16)), dim3(256), 0, s, at<float2>(ws, q.part), (long)n, cdiv(V, kTile),
                     at<float>(ws, q.zlab), labels, n, V, ignore, (float*)loss, (float*)lse);
  return (int)hipGetLastError();
}

template <typename T>
int backward(const void* h, long ldh, const void* w, long ldw, const float* bias, const int* labels, const float* lse,
             const float* row_scale, float grad_scale, int n, int H, int V, int ignore, int piece, void* dh, void* dw, int dw_f32,
             void* db, void* ws, hipStream_t s) {
  const int E = sizeof(T);
  const bool h_ok = rows_ok(h, ldh, H, E), w_ok = rows_ok(w, ldw, H, E);
  const Plan q = plan_for(E == 2 ? 1 : 0, 1, n, H, V, h_ok, w_ok, db != nullptr, piece);
  const void* hp = h;
  long ldhp = ldh;
  if (!h_ok) {
    VH_TRY(launch_pad((const T*)h, ldh, n, H, at<T>(ws, q.h_pad), q.ldk, s));
    hp = at<T>(ws, q.h_pad);
    ldhp = q.ldk;
  }
  VH_TRY(launch_transpose((const T*)h, ldh, n, H, at<T>(ws, q.hT), q.ldn, labels, ignore, s));
  for (int k = 0; k < q.pieces; ++k) {
    const int v0 = k * q.piece, vn = V - v0 < q.piece ? V - v0 : q.piece;
    const long ldv = up(vn, 64 / E);
    const T* wp = (const T*)w + (long)v0 * ldw;
    VhOperands p{wp, hp, ldw, ldhp, vn, n, (int)q.ldk, 0, 0};
    if (!w_ok) {
      VH_TRY(launch_pad(wp, ldw, vn, H, at<T>(ws, q.w_pad), q.ldk, s));
      p.A = at<T>(ws, q.w_pad);
      p.lda = q.ldk;
    }
    VhGradLogits e{bias ? bias + v0 : nullptr, labels, lse, row_scale, grad_scale, v0, V, ignore, at<T>(ws, q.d), ldv,
                   db ? at<float>(ws, q.dbpart) : nullptr};
    VH_TRY((run_gemm<T>(p, e, s)));
    if (db) {
      hipLaunchKernelGGL(vh_dbias, dim3(cdiv(vn, 256)), dim3(256), 0, s, at<float>(ws, q.dbpart), ldv, q.row_tiles, (float*)db + v0, vn);
      VH_TRY((int)hipGetLastError());
    }
    if (dw) {
      VH_TRY(launch_transpose((const T*)at<T>(ws, q.d), ldv, n, vn, at<T>(ws, q.dT), q.ldn, nullptr, 0, s));
      VhStore st{(char*)dw + (long)v0 * H * (dw_f32 ? 4 : E), H, dw_f32, nullptr, 1, 1};
      VH_TRY((run_gemm<T>(VhOperands{at<T>(ws, q.hT), at<T>(ws, q.dT), q.ldn, q.ldn, H, vn, (int)q.ldn, 0, 0}, st, s)));
    }
    if (dh) {
      VH_TRY(launch_transpose(wp, ldw, vn, H, at<T>(ws, q.wT), ldv, nullptr, 0, s));
      VhStore st{dh, H, 0, q.sum ? at<float>(ws, q.sum) : nullptr, k == 0, k == q.pieces - 1};
      VH_TRY((run_gemm<T>(VhOperands{at<T>(ws, q.wT), at<T>(ws, q.d), ldv, ldv, H, n, (int)ldv, 0, 0}, st, s)));
    }
  }
  return 0;
}

bool sizes_ok(int dtype, long n, int H, int V, long ldh, long ldw) {
  return (dtype == 0 || dtype == 1) && n > 0 && n <= kMaxRow && H > 0 && H <= kMaxRow && V > 0 && V < (1 << 30) && ldh >= H &&
         ldw >= H && ldh <= kMaxRow && ldw <= kMaxRow;
}

}  // namespace

extern "C" {

// dtype: 0 fp32, 1 bf16.  piece: classes per piece of the backward pass (0: the default).  Returns < 0 for bad arguments.
long dtf_vocab_head_workspace(int dtype, int backward_pass, const void* h, long ldh, const void* w, long ldw, int n, int H, int V,
                              int bias, int piece) {
  if (!sizes_ok(dtype, n, H, V, ldh, ldw) || piece < 0 || piece > kMaxRow) return -3;
  const int E = esize(dtype);
  return plan_for(dtype, backward_pass, n, H, V, rows_ok(h, ldh, H, E), rows_ok(w, ldw, H, E), bias != 0, piece).total;
}

// loss[n], lse[n] (fp32) of h [n][H] (rows ldh apart) against w [V][H] (rows ldw apart), bias [V] fp32 or NULL, labels int32
int dtf_vocab_head_fwd(int dtype, const void* h, long ldh, const void* w, long ldw, const void* bias, const void* labels, int n,
                       int H, int V, int ignore, void* loss, void* lse, void* ws, long ws_bytes, hipStream_t s) {
  if (!sizes_ok(dtype, n, H, V, ldh, ldw) || !h || !w || !labels || !loss || !lse || !ws || ((uintptr_t)ws & 255)) return -3;
  if ((uintptr_t)h & (esize(dtype) - 1) || (uintptr_t)w & (esize(dtype) - 1)) return -3;
  if (ws_bytes < dtf_vocab_head_workspace(dtype, 0, h, ldh, w, ldw, n, H, V, bias != nullptr, 0)) return -2;
  return dtype == 1 ? forward<bf16>(h, ldh, w, ldw, (const float*)bias, (const int*)labels, n, H, V, ignore, loss, lse, ws, s)
                    : forward<float>(h, ldh, w, ldw, (const float*)bias, (const int*)labels, n, H, V, ignore, loss, lse, ws, s);
}

// dh [n][H] in the operand type, dw [V][H] in the operand type or fp32 (dw_f32), db [V] fp32; each may be NULL (not wanted).
// d loss / d loss_i = grad_scale * row_scale[i] (row_scale fp32 [n] or NULL: 1)
int dtf_vocab_head_bwd(int dtype, const void* h, long ldh, const void* w, long ldw, const void* bias, const void* labels,
                       const void* lse, const void* row_scale, float grad_scale, int n, int H, int V, int ignore, int piece, void* dh,
                       void* dw, int dw_f32, void* db, void* ws, long ws_bytes, hipStream_t s) {
  if (!sizes_ok(dtype, n, H, V, ldh, ldw) || !h || !w || !labels || !lse || !ws || ((uintptr_t)ws & 255) || piece < 0 || piece > kMaxRow) return -3;
  if ((uintptr_t)h & (esize(dtype) - 1) || (uintptr_t)w & (esize(dtype) - 1) || ((uintptr_t)dh & 15) || ((uintptr_t)dw & 15)) return -3;
  if (ws_bytes < dtf_vocab_head_workspace(dtype, 1, h, ldh, w, ldw, n, H, V, db != nullptr, piece)) return -2;
  return dtype == 1 ? backward<bf16>(h, ldh, w, ldw, (const float*)bias, (const int*)labels, (const float*)lse, (const float*)row_scale,
                                     grad_scale, n, H, V, ignore, piece, dh, dw, dw_f32, db, ws, s)
                    : backward<float>(h, ldh, w, ldw, (const float*)bias, (const int*)labels, (const float*)lse, (const float*)row_scale,
                                      grad_scale, n, H, V, ignore, piece, dh, dw, dw_f32, db, ws, s);
}

}  // extern "C"
