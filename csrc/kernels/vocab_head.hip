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
// All products run through one kernel template, vh_gemm: out[j][i] = sum_k A(i, k) B(j, k), where an operand lies in memory
// with k contiguous (fast) or with its rows contiguous (slow); nothing is transposed in memory.
#include <type_traits>
#include "common.hpp"
#include "api.h"

namespace dtf {

constexpr float kLog2e = 1.4426950408889634f;
typedef f32x4 f32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ f32x4 vh_mma(const u32x4& a, const u32x4& b, f32x4 c) {
  return mfma16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}

// fp32 operands are multiplied on the bf16 matrix cores: a value is the sum of three bf16 values, each the leading 8 bits of what
// the ones before it leave (together all 24), products of two bf16 values are exact in the fp32 accumulators, and of the nine the
// three smallest are left out:
//   a b = a1 b1 + (a1 b2 + a2 b1) + (a1 b3 + a2 b2 + a3 b1) + at most 2^-21 |a b| (2^-23 on average)
// for values from about 2e-34 on; below, the third part ends at 2^-133, bf16's smallest step, and up to 2^-133 (|a| + |b|) is lost
// as well (of 1e-35 1e-5, of 1e-37 1e-3: an upstream gradient of a row, which is multiplied into d, may be as small; the common
// grad_scale is not).
// Six bf16 instructions do 16 x 16 x 32 in 96 cycles, the fp32 ones (16 x 16 x 4) take 256.  An infinite value gives NaN (its
// second part is inf - inf).  The leading bits are cut off, not rounded: the conversion instruction is several times slower than a
// mask and a byte permutation (4096 x 1024 x 16000 forward 605 and 567 us; with the fp32 instructions 971, 138 TFLOP/s of their
// 157).  ROUND: the first part is rounded (half a step added before the cut), so that what is left out has no sign of its own (at
// most 2^-22): one instruction more per value, for few rows, whose single losses show it (1 x 300 x 700, lse near its label's
// logit: loss off by 4.6e-6 of itself, 1.2e-6 with it).  Values that round beyond 3.39e38 count as infinite there.
struct VhSplit {
  u32x4 part[3];
};
template <bool ROUND>
__device__ __forceinline__ VhSplit vh_split(const u32x4& k0, const u32x4& k1) {
  const f32x4 x = __builtin_bit_cast(f32x4, k0), y = __builtin_bit_cast(f32x4, k1);
  float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  VhSplit s;
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const unsigned half = ROUND && q == 0 ? 0x8000u : 0u;
      const unsigned lo = __builtin_bit_cast(unsigned, v[e]) + half, hi = __builtin_bit_cast(unsigned, v[e + 1]) + half;
      s.part[q][e / 2] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
      v[e] -= __builtin_bit_cast(float, lo & 0xffff0000u);
      v[e + 1] -= __builtin_bit_cast(float, hi & 0xffff0000u);
    }
  return s;
}

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

// Buffer descriptor from values that are the same in every lane, said so: 64-bit address arithmetic is done on the vector
// units, and a descriptor that comes from there is otherwise taken lane by lane in a loop around every load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t vh_rsrc(const char* p, size_t bytes) {
  const uint64_t a = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  const uint32_t n = __builtin_amdgcn_readfirstlane((uint32_t)(bytes < 0x7ffffff0u ? bytes : 0x7ffffff0u));
  return make_rsrc((const void*)(((uint64_t)hi << 32) | lo), n);
}

struct VhOperands {
  // Fast operand: [rows][K], ld elements between rows, k contiguous.  Slow operand: [K][rows], ld elements between the K
  // rows.  Rows start on 4 bytes, 16-byte LDS-DMAs need no more; their descriptors are checked for every 4 bytes, so that no read
  // goes behind an operand.  What a fast operand's last 16 bytes of K hold behind K (its next row) meets zeros of the other one.
  const void *A, *B;
  long lda, ldb;
  int M, N, Ka, Kb;       // Ka, Kb: k from there on counts as zero
  int tiles_m, tiles_n;
  int ktiles, splits;     // K tiles of 128 bytes (of the operand type); workgroups that share a tile's K range
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
  int lane, wave, split;
};

// LDS-DMA of one operand's K tile (128 bytes of k for ROWS rows) and the fragment reads from it.
//   fast: LDS rows of 128 bytes; chunk (16 bytes) p of row r holds chunk p ^ (r & 7): a fragment read of 16 rows touches
//         every bank once.  A half tile is one 16-byte read per lane: group g holds the chunk g (bf16: k = 8 g .. 8 g + 7,
//         fp32: k = 4 g .. 4 g + 3).
//   slow: LDS rows are the K rows, ROWS elements long; the 16-element windows of a row are permuted by row.  bf16 fragments
//         come from transposed reads, two per fragment, which give group g the k = 4 g .. 4 g + 3 and 16 + 4 g .. + 3 of the
//         half; fp32 ones from four 4-byte reads, k = 4 g .. 4 g + 3 as in a fast operand.
// What a slow operand's window numbers are XORed with (bf16: eight rows of a transposed read in eight windows, or two rows to
// the 256 bytes of all banks where a row is 128 bytes; fp32: the four groups of a read).
template <int E, int ROWB>
__device__ __forceinline__ int vh_window_key(int row) {
  return E == 2 ? (ROWB >= 256 ? row & 7 : (row >> 1) & 3) : (row >> 2) & 3;
}
template <typename T, int ROWS, bool SLOW, int NT>
struct VhLoader {
  static constexpr int E = sizeof(T), KT = 128 / E, CH = ROWS * 8 / NT, CPR = ROWS * E / 16, ROWB = ROWS * E;
  static_assert(ROWS * 8 % NT == 0 && (!SLOW || NT % CPR == 0), "every thread stages whole chunks");
  const char* base;
  long ld;
  uint32_t v0, step;
  int K, rows, kch;

  __device__ __forceinline__ void init(const void* p, long ld_, int r0, int total, int K_, int tid) {
    ld = ld_ * E;
    K = K_;
    rows = total - r0;
    if (SLOW) {
      rows = (rows + 4 / E - 1) & ~(4 / E - 1);        // whole words: an odd number of bf16 values is padded
      base = (const char*)p + (size_t)r0 * E;
    } else {
      base = (const char*)p + (size_t)r0 * ld;
      kch = ((tid & 7) ^ ((tid >> 3) & 7)) << 4;       // the same for every chunk of a thread: NT is a multiple of 64
      v0 = (uint32_t)(tid >> 3) * (uint32_t)ld + kch;
      step = (uint32_t)(NT / 8) * (uint32_t)ld;
    }
  }
  static __device__ __forceinline__ int key(int row) { return vh_window_key<E, ROWB>(row) * (E == 2 ? 2 : 4); }
  // lds: start of this operand's part of the buffer
  __device__ __forceinline__ void dma(int t, char* lds, int wave, int tid) const {
    char* const dst = lds + wave * 1024;
    if constexpr (SLOW) {
      const int left = K - t * KT;
      const size_t bytes = left > 0 ? (size_t)(left - 1) * ld + (size_t)rows * E : 0;
      const __amdgpu_buffer_rsrc_t r = vh_rsrc(base + (size_t)t * KT * ld, bytes);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int q = tid + i * NT, row = q / CPR, ch = q % CPR;
        vh_dma16(r, dst + i * NT * 16, (uint32_t)row * (uint32_t)ld + ((ch ^ key(row)) << 4), 0);
      }
    } else {
      const uint32_t so = (uint32_t)t << 7;
      const int n = rows < ROWS ? rows : ROWS;
      const __amdgpu_buffer_rsrc_t r = vh_rsrc(base, (size_t)(n - 1) * ld + (size_t)K * E);
      // K may end inside the tile: zeros from there on (an offset behind every descriptor: tiles span less than 2 GB)
      const uint32_t v = (int)so + kch < K * E ? v0 : 0x80000000u;
#pragma unroll
      for (int i = 0; i < CH; ++i) vh_dma16(r, dst + i * NT * 16, v + i * step, so);
    }
  }
};

// fragments of 16 rows r0 .. r0 + 15 (+ 16 i) from an operand's LDS part, half 0 or 1 of the K tile
template <typename T, int ROWS, bool SLOW, int CNT>
struct VhFrags {
  static constexpr int E = sizeof(T), ROWB = ROWS * E;
  int off;
  __device__ __forceinline__ void init(int r0, int lane) {
    const int i16 = lane & 15, g = lane >> 4;
    if (!SLOW) off = (r0 + i16) * 128 + ((g ^ (i16 & 7)) << 4);
    else if (E == 2) off = (4 * g + (i16 >> 2)) * ROWB + (((r0 >> 4) ^ vh_window_key<E, ROWB>(4 * g + (i16 >> 2))) << 5) + 8 * (i16 & 3);
    else off = 4 * g * ROWB + (((r0 >> 4) ^ vh_window_key<E, ROWB>(4 * g)) << 6) + 4 * i16;
  }
  __device__ __forceinline__ u32x4 one(const char* lds, int half, int i) const {
    static_assert(!SLOW || E == 4, "bf16 slow operands are read by read_tr");
    if constexpr (!SLOW) {
      return *reinterpret_cast<const u32x4*>(lds + (off ^ (half << 6)) + i * 2048);
    } else {
      u32x4 f;
#pragma unroll
      for (int s = 0; s < 4; ++s) f[s] = *reinterpret_cast<const unsigned*>(lds + half * 16 * ROWB + (off ^ (i << 6)) + s * ROWB);
      return f;
    }
  }
  __device__ __forceinline__ void read(u32x4 (&f)[CNT], const char* lds, int half) const {
#pragma unroll
    for (int i = 0; i < CNT; ++i) f[i] = one(lds, half, i);
  }
  // Fragments i .. i + 3 (or both of CNT == 2) of a bf16 slow operand.  The reads and the wait for them are one block: nothing
  // between them can use, move or reuse a register that is still being written.
  static constexpr int TR = CNT < 4 ? CNT : 4;
  __device__ __forceinline__ void read_tr(u32x4* f, const char* lds, int half, int i) const {
    const uint32_t p = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)(const void*)(lds + half * 32 * ROWB);
    const uint32_t a0 = p + (off ^ (i << 5)), a1 = p + (off ^ ((i + 1) << 5));
    u32x2 w0, w1, x0, x1;
    if constexpr (TR == 4) {
      const uint32_t a2 = p + (off ^ ((i + 2) << 5)), a3 = p + (off ^ ((i + 3) << 5));
      u32x2 y0, y1, z0, z1;
      asm volatile(
          "ds_read_b64_tr_b16 %0, %8\n\t"
          "ds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
          "ds_read_b64_tr_b16 %2, %9\n\t"
          "ds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
          "ds_read_b64_tr_b16 %4, %10\n\t"
          "ds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
          "ds_read_b64_tr_b16 %6, %11\n\t"
          "ds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(w0), "=&v"(w1), "=&v"(x0), "=&v"(x1), "=&v"(y0), "=&v"(y1), "=&v"(z0), "=&v"(z1)
          : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(16 * ROWB)
          : "memory");
      f[2] = (u32x4){y0[0], y0[1], y1[0], y1[1]};
      f[3] = (u32x4){z0[0], z0[1], z1[0], z1[1]};
    } else {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %4\n\t"
          "ds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
          "ds_read_b64_tr_b16 %2, %5\n\t"
          "ds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(w0), "=&v"(w1), "=&v"(x0), "=&v"(x1)
          : "v"(a0), "v"(a1), "n"(16 * ROWB)
          : "memory");
    }
    f[0] = (u32x4){w0[0], w0[1], w1[0], w1[1]};
    f[1] = (u32x4){x0[0], x0[1], x1[0], x1[1]};
  }
};

// Main loop: K tiles t0 .. t1 - 1 in D LDS buffers (two for the large tiles, which take all of LDS; four for small ones, whose
// tiles are over sooner than their operands arrive).
//
// bf16, both operands fast: a tile is multiplied in two halves, and the fragments of a half are read during the MFMAs of
// the half before it, one barrier per tile:
//   read the second half of tile t | MFMAs on the first | wait until tile t + 1 has landed, barrier
//   DMA of tile t + D into the buffer of tile t | read the first half of tile t + 1 | MFMAs on the second half of tile t
// fp32, and a bf16 slow operand (fragments are read, fp32 ones split, right before their MFMAs; the other wave of the SIMD covers
// that):
//   wait until tile t has landed, barrier | DMA of tile t + D - 1 into the buffer of tile t - 1 | both halves of tile t
//
// The epilogue's inputs (labels, log-sum-exps, biases of the tile) are requested before the first operand tile and put into
// LDS behind it, where they cost no latency at the end.
template <typename T, int BM, int BN, int NWM, int NWN, bool AS, bool BS, int D, class Epi, class Tile>
__device__ __forceinline__ void vh_mainloop(const VhOperands& p, Tile& c, char* lds, int t0, int t1, const Epi& e,
                                            typename Epi::template Inputs<BM, BN>* in) {
  constexpr int NT = Tile::NT, MT = Tile::MT, NTL = Tile::NTL;
  constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128;
  typedef VhLoader<T, BM, AS, NT> LA;
  typedef VhLoader<T, BN, BS, NT> LB;
  constexpr int NDMA = LA::CH + LB::CH;
  const int tid = threadIdx.x;
  LA la;
  LB lb;
  la.init(p.A, p.lda, c.m0, p.M, p.Ka, tid);
  lb.init(p.B, p.ldb, c.n0, p.N, p.Kb, tid);
  VhFrags<T, BM, AS, MT> ra;
  VhFrags<T, BN, BS, NTL> rb;
  ra.init(c.wm0, c.lane);
  rb.init(c.wn0, c.lane);
  auto dma = [&](int t, char* buf) {
    la.dma(t, buf, c.wave, tid);
    lb.dma(t, buf + ABYTES, c.wave, tid);
  };
  char* const ring_end = lds + D * STAGE;
  auto next = [&](char* buf) { return buf + STAGE == ring_end ? lds : buf + STAGE; };
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NTL; ++j) c.acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if (t0 >= t1) return;
  const auto early = e.template request<BM, BN, NT>(p, c.m0, c.n0, tid);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int d = 0; d + 1 < D; ++d)
      if (t0 + d < t1) dma(t0 + d, lds + d * STAGE);
    e.template keep<BM, BN, NT>(early, in, tid);
    char* buf = lds;
    char* last = lds + (D - 1) * STAGE;         // the buffer of tile t - 1
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      if (D > 2 && t + D - 1 <= t1) vh_wait<(D - 2) * NDMA>();
      else vh_wait<0>();
      vh_barrier();
      if (t + D - 1 < t1) dma(t + D - 1, last);
      // Few rows' logits: a K tile is summed by itself and then added, one rounding of the long sum instead of six (3 rows, 3883 x
      // 3931: losses off by up to 2.0e-6 of themselves, 3.9e-7 with it; 100 rows, 1024 x 10000: 3.4e-7 and 8.6e-8).  Large tiles
      // have no room for it among their vector instructions.
      constexpr bool FEW = MT * NTL <= 4;
      VhSplit b[NTL];
#pragma unroll
      for (int j = 0; j < NTL; ++j) b[j] = vh_split<FEW>(rb.one(buf + ABYTES, 0, j), rb.one(buf + ABYTES, 1, j));
      VhSplit a = vh_split<FEW>(ra.one(buf, 0, 0), ra.one(buf, 1, 0));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        constexpr int TERMS[6][2] = {{0, 2}, {2, 0}, {1, 1}, {0, 1}, {1, 0}, {0, 0}};      // the smallest first
        VhSplit ahead = a;
        if (i + 1 < MT) ahead = vh_split<FEW>(ra.one(buf, 0, i + 1), ra.one(buf, 1, i + 1));
        f32x4 sum[NTL];
#pragma unroll
        for (int j = 0; j < NTL; ++j) sum[j] = FEW ? (f32x4){0.f, 0.f, 0.f, 0.f} : c.acc[i][j];
#pragma unroll
        for (int q = 0; q < 6; ++q)
#pragma unroll
          for (int j = 0; j < NTL; ++j) sum[j] = vh_mma(a.part[TERMS[q][0]], b[j].part[TERMS[q][1]], sum[j]);
#pragma unroll
        for (int j = 0; j < NTL; ++j) c.acc[i][j] = FEW ? c.acc[i][j] + sum[j] : sum[j];
        a = ahead;
        // the next fragment (44 vector instructions) is split in the shadow of this one's MFMAs, behind the first two, while it
        // arrives (4096 x 1024 x 16000 forward, 7 % less)
        if (i + 1 < MT) {
          constexpr int PER = (44 + 6 * NTL - 3) / (6 * NTL - 2);
          __builtin_amdgcn_sched_group_barrier(0x100, AS ? 8 : 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
#pragma unroll
          for (int x = 2; x < 6 * NTL; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, PER, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      last = buf;
      buf = next(buf);
    }
  } else if constexpr (AS || BS) {
    typedef VhFrags<T, BM, AS, MT> RA;
    typedef VhFrags<T, BN, BS, NTL> RB;
    static_assert(AS && MT % RA::TR == 0 && (!BS || NTL % RB::TR == 0), "slow products: dh (A) and dw (A and B)");
#pragma unroll
    for (int d = 0; d + 1 < D; ++d)
      if (t0 + d < t1) dma(t0 + d, lds + d * STAGE);
    e.template keep<BM, BN, NT>(early, in, tid);
    u32x4 fb[2][NTL];
    char* buf = lds;
    char* last = lds + (D - 1) * STAGE;         // the buffer of tile t - 1
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      if (D > 2 && t + D - 1 <= t1) vh_wait<(D - 2) * NDMA>();
      else vh_wait<0>();
      vh_barrier();
      if constexpr (!BS) rb.read(fb[0], buf + ABYTES, 0);
      if (t + D - 1 < t1) dma(t + D - 1, last);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (BS) {
#pragma unroll
          for (int j = 0; j < NTL; j += RB::TR) rb.read_tr(&fb[0][j], buf + ABYTES, h, j);
        } else if (h == 0) {
          rb.read(fb[1], buf + ABYTES, 1);
        }
#pragma unroll
        for (int i = 0; i < MT; i += RA::TR) {
          u32x4 a[RA::TR];
          ra.read_tr(a, buf, h, i);
#pragma unroll
          for (int k = 0; k < RA::TR; ++k)
#pragma unroll
            for (int j = 0; j < NTL; ++j) c.acc[i + k][j] = vh_mma(a[k], fb[BS ? 0 : h][j], c.acc[i + k][j]);
        }
      }
      last = buf;
      buf = next(buf);
    }
  } else {
    u32x4 fa[2][MT], fb[2][NTL];
    auto frags = [&](int x, const char* buf, int half) {
      ra.read(fa[x], buf, half);
      rb.read(fb[x], buf + ABYTES, half);
    };
    auto mma = [&](int x) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) c.acc[i][j] = vh_mma(fa[x][i], fb[x][j], c.acc[i][j]);
    };
    // the schedule of a half: the DMAs one MFMA apart, then the fragment reads spread over the others
    constexpr int R = MT + NTL, X = MT * NTL;
    constexpr int PER = (X - NDMA) / R > 0 ? (X - NDMA) / R : 1;
    auto spread = [&](bool dmas) {
      if (dmas) {
#pragma unroll
        for (int i = 0; i < NDMA; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (t0 + d < t1) dma(t0 + d, lds + d * STAGE);
    e.template keep<BM, BN, NT>(early, in, tid);
    if (t0 + D <= t1) vh_wait<(D - 1) * NDMA>();
    else vh_wait<0>();
    vh_barrier();
    frags(0, lds, 0);
    vh_wait<63>();
    int t = t0;
    char* buf = lds;
#pragma unroll 1
    for (; t + D < t1; ++t) {
      frags(1, buf, 1);
      mma(0);
      spread(false);
      vh_wait<(D - 2) * NDMA>();
      vh_barrier();
      dma(t + D, buf);
      buf = next(buf);
      frags(0, buf, 0);
      mma(1);
      spread(true);
      vh_wait<63>();
    }
#pragma unroll 1
    for (; t < t1; ++t) {
      frags(1, buf, 1);
      mma(0);
      vh_wait<0>();
      vh_barrier();
      buf = next(buf);
      frags(0, buf, 0);      // (behind the last tile: some buffer, read and not used)
      mma(1);
      vh_wait<63>();
    }
  }
  vh_wait<0>();
  vh_barrier();
}

// dst[r][c] = src[r][c], r < R, with rows ldd apart (16-byte multiples), columns C .. ldd - 1 zero and rows from `rows` on zero.
// labels given: the rows of ignored labels are zero as well -- whatever lies there, 0 * NaN must not reach a gradient.  Whole
// 16-byte chunks from any element of a row (global memory takes unaligned vector loads), the last chunk of a row element by
// element.  twin: elements to a second copy (0: none).
struct VhCopy {
  const void* src;
  long lds_;
  int R, rows, C;
  void* dst;
  long ldd;
  const int* labels;
  int ignore;
  long twin;
  int blocks;           // workgroups that do this besides a product (0: a launch of its own)
};
template <typename T>
__device__ __forceinline__ void vh_copy_rows(const VhCopy& c, long first, long step) {
  constexpr int V = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(V))) T vec;
  typedef vec vec_any __attribute__((aligned(sizeof(T))));
  const int per = (int)(c.ldd / V);
  const long n = (long)c.R * per;
  for (long x = first; x < n; x += step) {
    const long r = n >> 32 ? x / per : (long)((unsigned)x / (unsigned)per);
    const int i = (int)(x - r * per) * V;
    vec v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)0.f;
    if (r < c.rows && !(c.labels && c.labels[r] == c.ignore)) {
      const T* p = (const T*)c.src + r * c.lds_ + i;
      if (i + V <= c.C) {
        const vec y = *reinterpret_cast<const vec_any*>(p);
        v = y;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i + e < c.C) v[e] = p[e];
      }
    }
    T* const o = (T*)c.dst + r * c.ldd + i;
    *reinterpret_cast<vec*>(o) = v;
    if (c.twin) *reinterpret_cast<vec*>(o + c.twin) = v;
  }
}

// Which tile and which split a workgroup takes.  Workgroups are dealt round-robin over the 8 XCDs; each XCD gets one run of the
// (split, band of four tile rows, column) order, so that its L2 serves all tiles of a split from one fetch of the split's
// operands.
__device__ __forceinline__ int vh_assign(int L, int gx, int gy, int splits, int& tx, int& ty) {
  constexpr int NX = 8, BH = 4;
  const int tiles = gx * gy, total = tiles * splits, xcd = L % NX, q = total / NX, r = total % NX;
  int idx = xcd * q + min(xcd, r) + L / NX;
  const int split = idx / tiles;
  idx -= split * tiles;
  const int band = idx / (BH * gx), rem = idx - band * BH * gx, h = min(BH, gy - band * BH);
  tx = rem / h;
  ty = band * BH + rem % h;
  return split;
}

template <typename T, int BM, int BN, int NWM, int NWN, bool AS, bool BS, int D, class Epi>
__global__ __launch_bounds__(NWM * NWN * 64, 1) void vh_gemm(VhOperands p, Epi e) {
  typedef VhTile<T, BM, BN, NWM, NWN> Tile;
  // one LDS object: with two of them the compiler orders every fragment read behind all LDS-DMAs in flight (s_waitcnt
  // vmcnt(0) in the middle of the loop, forward 15 % slower)
  typedef typename Epi::template Inputs<BM, BN> Inputs;
  __shared__ __attribute__((aligned(16))) char lds[D * (BM + BN) * 128 + sizeof(Inputs)];
  Inputs& in = *reinterpret_cast<Inputs*>(lds + D * (BM + BN) * 128);
  if constexpr (Epi::kCopies) {         // the workgroups behind the tiles
    const int tiles = p.tiles_m * p.tiles_n * p.splits;
    if ((int)blockIdx.x >= tiles) {
      vh_copy_rows<T>(e.copy, (long)(blockIdx.x - tiles) * Tile::NT + threadIdx.x, (long)e.copy.blocks * Tile::NT);
      return;
    }
  }
  Tile c;
  c.lane = threadIdx.x & 63;
  c.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  c.wm0 = (c.wave / NWN) * Tile::WM;
  c.wn0 = (c.wave % NWN) * Tile::WN;
  int tx, ty;
  c.split = vh_assign(blockIdx.x, p.tiles_m, p.tiles_n, p.splits, tx, ty);
  c.m0 = tx * BM;
  c.n0 = ty * BN;
  const int per = (p.ktiles + p.splits - 1) / p.splits, t0 = c.split * per;
  vh_mainloop<T, BM, BN, NWM, NWN, AS, BS, D>(p, c, lds, t0, min(p.ktiles, t0 + per), e, &in);
  e.template run<T, BM, BN, NWM, NWN>(p, c, tx, ty, lds, in);
}

// ---- epilogues ------------------------------------------------------------------------------------------------------
// Inputs of the logits' epilogues, per row and per class of the tile
struct VhRowInputs {
  int label;          // relative to the tile's first class; never a class of the tile where the row has none there
  float l2, sc;       // base-2 log-sum-exp and upstream gradient (backward)
};
template <int BM, int BN>
struct VhLogitsInputs {
  VhRowInputs row[BN];
  float bias[BM];     // -inf for classes beyond the last one
};
template <int BM, int BN, int NT>
struct VhEarly {
  VhRowInputs row[(BN + NT - 1) / NT];
  float bias[(BM + NT - 1) / NT];
};
template <class Epi, int BM, int BN, int NT>
__device__ __forceinline__ VhEarly<BM, BN, NT> vh_request(const Epi& e, const VhOperands& p, int m0, int n0, int tid) {
  VhEarly<BM, BN, NT> x;
#pragma unroll
  for (int k = 0; k < (BN + NT - 1) / NT; ++k) {
    const int j = tid + k * NT;
    x.row[k] = j < BN && n0 + j < p.N ? e.row_inputs(n0 + j, m0) : VhRowInputs{-1, 0.f, 0.f};
  }
#pragma unroll
  for (int k = 0; k < (BM + NT - 1) / NT; ++k) {
    const int i = tid + k * NT;
    x.bias[k] = i < BM && m0 + i < p.M ? (e.bias ? e.bias[m0 + i] : 0.f) : -INFINITY;
  }
  return x;
}
template <int BM, int BN, int NT>
__device__ __forceinline__ void vh_keep(const VhEarly<BM, BN, NT>& x, VhLogitsInputs<BM, BN>* in, int tid) {
#pragma unroll
  for (int k = 0; k < (BN + NT - 1) / NT; ++k)
    if (tid + k * NT < BN) in->row[tid + k * NT] = x.row[k];
#pragma unroll
  for (int k = 0; k < (BM + NT - 1) / NT; ++k)
    if (tid + k * NT < BM) in->bias[tid + k * NT] = x.bias[k];
}
// acc += bias, and -inf beyond the last class; nothing to do inside a product without a bias
template <class Tile, int BM, int BN>
__device__ __forceinline__ void vh_add_bias(Tile& c, const VhLogitsInputs<BM, BN>& in, bool any, int M) {
  if (!any && c.m0 + BM <= M) return;
#pragma unroll
  for (int i = 0; i < Tile::MT; ++i) {
    const f32x4 b = *reinterpret_cast<const f32x4*>(&in.bias[c.wm0 + 16 * i + 4 * (c.lane >> 4)]);
#pragma unroll
    for (int j = 0; j < Tile::NTL; ++j) c.acc[i][j] += b;
  }
}

// Place of class k (0 .. 31) among the 32 of its group in a row of d: bf16 products read d with contiguous k next to a slow
// operand whose transposed reads deliver k = 4 g .. 4 g + 3 and 16 + 4 g .. + 3 to lane group g, so those eight lie together.
__device__ __forceinline__ int vh_place(int k) { return (k & ~31) | ((k & 12) << 1) | ((k & 16) >> 2) | (k & 3); }
__device__ __forceinline__ int vh_class(int at) { return (at & ~31) | ((at & 24) >> 1) | ((at & 4) << 2) | (at & 3); }

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
  static constexpr bool kCopies = false;
  const float* bias;
  const int* labels;
  int c0;                   // the product's first class
  float2* part;
  float* zlab;
  long ldpart;
  template <int BM, int BN> using Inputs = VhLogitsInputs<BM, BN>;
  __device__ __forceinline__ VhRowInputs row_inputs(int row, int m0) const {
    const int y = labels[row];
    return {y < c0 ? -1 : y - c0 - m0, 0.f, 0.f};
  }
  template <int BM, int BN, int NT>
  __device__ __forceinline__ VhEarly<BM, BN, NT> request(const VhOperands& p, int m0, int n0, int tid) const {
    return vh_request<VhForward, BM, BN, NT>(*this, p, m0, n0, tid);
  }
  template <int BM, int BN, int NT>
  __device__ __forceinline__ void keep(const VhEarly<BM, BN, NT>& x, VhLogitsInputs<BM, BN>* in, int tid) const {
    vh_keep<BM, BN, NT>(x, in, tid);
  }
  template <typename T, int BM, int BN, int NWM, int NWN, class Tile>
  __device__ __forceinline__ void run(const VhOperands& p, Tile& c, int tx, int, char* lds, const Inputs<BM, BN>& in) const {
    constexpr int MT = Tile::MT, NTL = Tile::NTL;
    const int i16 = c.lane & 15, g = c.lane >> 4;
    MaxSum (*red)[BN] = reinterpret_cast<MaxSum(*)[BN]>(lds);
    vh_add_bias(c, in, bias != nullptr, p.M);
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
      const int jl = c.wn0 + 16 * j + i16;
      const int y = in.row[jl].label - (c.wm0 + 4 * g);      // label relative to this lane's first class
      if (__any(y >= 0 && y < Tile::WM)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (y == 16 * i + r) zlab[c.n0 + jl] = c.acc[i][j][r];
      }
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, c.acc[i][j][r]);
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float m2 = m * kLog2e, off = m == -INFINITY ? 0.f : m2;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          s0 += __builtin_amdgcn_exp2f(fmaf(c.acc[i][j][r], kLog2e, -off));
          s1 += __builtin_amdgcn_exp2f(fmaf(c.acc[i][j][r + 1], kLog2e, -off));
        }
      float s = s0 + s1;
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if (g == 0) red[c.wave / NWN][jl] = {m2, s};
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

// Backward, first product: i = class (relative to the piece), j = row.  d[row][vh_place(class)], places up to ldd (a multiple
// of the K tile) written as zeros; dbias partial sums per row tile from the values before rounding.
// d is rounded to the operand type because the two products that read it multiply in that type: at most half a step of each
// value, summed in fp32.  The common factor grad_scale is left to those products' epilogues: 1/n times a label's -(1 - p), the
// value that outweighs all others of its row and class, would be rounded the same way for every row.  With up to 32 rows, half
// a tile of them, the rounding errors themselves are kept as rows 32 to 63, next to nothing in time: one row's gradient is then as
// exact as if d had stayed in fp32 (one row: 0.17 % rms, the operand type's own rounding, instead of up to 0.4; 16 rows, 4096 x
// 32000, backward 161 -> 166 us.  For 64 rows, a second tile, it would be 168 -> 211 us, and errors of many rows even out.)
// KEEP: more rows keep them, too, behind d, and dh and dw are products of both, for a caller who asks for it (4096 x 1024 x 65536:
// backward 1547 -> 2694 us, dw in fp32 off by 1.4e-6 rms instead of 8.7e-4).
template <bool KEEP>
struct VhGradLogitsT {
  static constexpr bool kCopies = true;
  VhCopy copy;              // h for dw: does not depend on d and needs no launch of its own
  const float* bias;        // of the piece
  const int* labels;
  const float* lse;
  const float* row_scale;   // or nullptr
  int v0, classes, ignore;  // the product's first class, all classes
  void* d;
  long ldd, rest;           // elements from a row to the row of its rounding errors (0: not kept; else, without KEEP, rows up to 32
                            // are written)
  int places;               // of this product's classes: up to there d is written
  float* dbpart;            // [row tile][ldd] or nullptr
  int dbplaces;             // up to there it is written
  float dbscale;
  template <int BM, int BN> using Inputs = VhLogitsInputs<BM, BN>;
  __device__ __forceinline__ VhRowInputs row_inputs(int row, int m0) const {
    const int y = labels[row];
    if (y == ignore) return {-1, 0.f, 0.f};
    const bool known = y >= 0 && y < classes;
    const float sc = row_scale ? row_scale[row] : 1.f;
    // (a label that is no class: the whole row says so)
    return {known && y >= v0 ? y - v0 - m0 : -1, lse[row] * kLog2e, known ? sc : __builtin_nanf("")};
  }
  template <int BM, int BN, int NT>
  __device__ __forceinline__ VhEarly<BM, BN, NT> request(const VhOperands& p, int m0, int n0, int tid) const {
    return vh_request<VhGradLogitsT, BM, BN, NT>(*this, p, m0, n0, tid);
  }
  template <int BM, int BN, int NT>
  __device__ __forceinline__ void keep(const VhEarly<BM, BN, NT>& x, VhLogitsInputs<BM, BN>* in, int tid) const {
    vh_keep<BM, BN, NT>(x, in, tid);
  }
  template <typename T, int BM, int BN, int NWM, int NWN, class Tile>
  __device__ __forceinline__ void run(const VhOperands& p, Tile& c, int, int ty, char* lds, const Inputs<BM, BN>& in) const {
    constexpr int MT = Tile::MT, NTL = Tile::NTL;
    constexpr bool REST = sizeof(T) == 2 && BM == 64;        // (the few rows' tiles)
    static_assert(!REST || MT % 2, "the single-fragment branch stores the errors");
    const int i16 = c.lane & 15, g = c.lane >> 4;
    const int mw = c.m0 + c.wm0 + 4 * g;
    vh_add_bias(c, in, bias != nullptr, p.M);
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
      const int jl = c.wn0 + 16 * j + i16, row = c.n0 + jl;
      const bool live = row < (!KEEP && REST && rest ? 32 : p.N);
      const VhRowInputs x = in.row[jl];
      const int y = x.label - (c.wm0 + 4 * g);
      const bool hit = y >= 0 && y < Tile::WM, dead = x.sc == 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) c.acc[i][j][r] = x.sc * __builtin_amdgcn_exp2f(fmaf(c.acc[i][j][r], kLog2e, -x.l2));
      if (__any(hit)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) c.acc[i][j][r] -= y == 16 * i + r ? x.sc : 0.f;
      }
      if (__any(dead)) {        // an ignored row is zero whatever its logits are (0 * inf and 0 * NaN are not)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) c.acc[i][j][r] = dead ? 0.f : c.acc[i][j][r];
      }
      if (live) {
        T* const o = (T*)d + (long)row * ldd;
        if constexpr (sizeof(T) == 2 && MT % 2 == 0) {      // eight neighbouring places: classes 4 g .. and 16 + 4 g ..
#pragma unroll
          for (int i = 0; i < MT; i += 2) {
            const int m = mw + 16 * i;
            const f32x4 v = c.acc[i][j], x = c.acc[i + 1][j];
            const bf16x8 y = {(T)v[0], (T)v[1], (T)v[2], (T)v[3], (T)x[0], (T)x[1], (T)x[2], (T)x[3]};
            if (m < places) {
              *reinterpret_cast<bf16x8*>(o + vh_place(m)) = y;
              if constexpr (KEEP) {
                bf16x8 left;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  left[r] = (T)(v[r] - (float)y[r]);
                  left[4 + r] = (T)(x[r] - (float)y[4 + r]);
                }
                *reinterpret_cast<bf16x8*>(o + vh_place(m) + rest) = left;
              }
            }
          }
        } else {
          typedef __attribute__((ext_vector_type(4))) T T4;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int m = mw + 16 * i;
            const f32x4 v = c.acc[i][j];
            const T4 y = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
            if (m >= places) continue;
            T* const at = o + (sizeof(T) == 2 ? vh_place(m) : m);
            *reinterpret_cast<T4*>(at) = y;
            if (REST && rest) *reinterpret_cast<T4*>(at + rest) = (T4){(T)(v[0] - (float)y[0]), (T)(v[1] - (float)y[1]),
                                                               (T)(v[2] - (float)y[2]), (T)(v[3] - (float)y[3])};
          }
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
      if (c.m0 + i < dbplaces) dbpart[(long)ty * ldd + c.m0 + i] = s * dbscale;
    }
  }
};

// Plain product: out[j][i], j < rows, in the operand type or fp32; the product's j is a place of d where by_place is set
// (its N is then the number of places).  With sum: fp32 [split][rows][M] running sums over the pieces of the classes, read
// unless `first` and written unless `last` (a single split: the last piece's result goes to out).  ONCE: the result is not to
// be kept in the caches (a template argument: as a value the compiler folds the two kinds of stores into the plain one).
template <bool ONCE>
struct VhStoreT {
  static constexpr bool kCopies = false;
  void* out;
  long ldo;
  int out_f32;
  int by_place;
  int rows;
  float* sum;
  int first, last;
  float scale;              // of what goes to out
  int fold;                 // rows 32 to 63 are added to 0 to 31
  // V values of a row, from the wave's staging rows to where they belong
  template <typename T, int V>
  __device__ __forceinline__ void put(const float* src, long row, int m, int M, int split) const {
    float v[V];
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(src + q);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[q + r] = x[r];
    }
    const bool whole = m + V <= M;
    if (sum) {
      float* s = sum + ((long)split * rows + row) * M + m;
      if (!first) {
#pragma unroll
        for (int q = 0; q < V; q += 4) {
          if (whole) {
            const f32x4 x = *reinterpret_cast<const f32x4_any*>(s + q);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[q + r] += x[r];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (m + q + r < M) v[q + r] += s[q + r];
          }
        }
      }
      if (!last) {
        store<float, V, false>(s, v, M - m);      // (read again soon)
        return;
      }
    }
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] *= scale;
    if (out_f32 || sizeof(T) == 4) store<float, V, ONCE>((float*)out + row * ldo + m, v, M - m);
    else store<T, V, ONCE>((T*)out + row * ldo + m, v, M - m);
  }
  template <typename O, int V, bool KEEP_OUT>
  static __device__ __forceinline__ void store(O* o, const float (&v)[V], int left) {
    constexpr int W = 16 / sizeof(O) < V ? 16 / sizeof(O) : V;
    typedef __attribute__((ext_vector_type(W))) O vec;
    typedef vec vec_any __attribute__((aligned(sizeof(O))));
    if (left >= V) {
#pragma unroll
      for (int q = 0; q < V; q += W) {
        vec x;
#pragma unroll
        for (int r = 0; r < W; ++r) x[r] = (O)v[q + r];
        if constexpr (KEEP_OUT) __builtin_nontemporal_store(x, reinterpret_cast<vec_any*>(o + q));
        else *reinterpret_cast<vec_any*>(o + q) = x;
      }
    } else {
#pragma unroll
      for (int r = 0; r < V; ++r)
        if (r < left) o[r] = (O)v[r];
    }
  }
  // A lane of the product holds four values of a row, sixteen rows side by side: stores of it would touch sixteen lines for
  // 32 or 64 bytes each.  Sixteen rows at a time go through a part of LDS of the wave's own and leave as whole runs of WM
  // values (16 rows x 132 floats: the 16-byte writes of a column group spread over all banks).
  struct None {};
  template <int BM, int BN> using Inputs = None;
  template <int BM, int BN, int NT>
  __device__ __forceinline__ None request(const VhOperands&, int, int, int) const { return {}; }
  template <int BM, int BN, int NT>
  __device__ __forceinline__ void keep(None, None*, int) const {}
  template <typename T, int BM, int BN, int NWM, int NWN, class Tile>
  __device__ __forceinline__ void run(const VhOperands& p, Tile& c, int, int, char* lds, const None&) const {
    constexpr int MT = Tile::MT, NTL = Tile::NTL, WM = Tile::WM, PITCH = WM + 4;
    constexpr int V = sizeof(T) == 2 ? 8 : 4, LPR = WM / V, RPP = 64 / LPR;       // lanes per row, rows per pass
    static_assert(NWM * NWN * 16 * PITCH * 4 <= 2 * (BM + BN) * 128, "staging rows fit in the tile buffers");
    float* const st = reinterpret_cast<float*>(lds) + c.wave * 16 * PITCH;
    const int i16 = c.lane & 15, g = c.lane >> 4;
    const int rl = c.lane / LPR, cl = (c.lane % LPR) * V, m = c.m0 + c.wm0 + cl;
    if constexpr (sizeof(T) == 2 && NWN == 1 && NTL == 4) {       // (the few rows' dh)
      if (fold)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) c.acc[i][j] += c.acc[i][j + 2];
    }
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
#pragma unroll
      for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(st + i16 * PITCH + 16 * i + 4 * g) = c.acc[i][j];
      asm volatile("" ::: "memory");        // other lanes' values are read: LDS accesses of a wave stay in this order
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r = 0; r < 16; r += RPP) {
        int row = c.n0 + c.wn0 + 16 * j + r + rl;
        if (sizeof(T) == 2 && by_place) row = vh_class(row);
        if (row < rows && m < p.M) put<T, V>(st + (r + rl) * PITCH + cl, row, m, p.M, c.split);
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
  }
};

typedef VhStoreT<false> VhStore;

// ---- small kernels --------------------------------------------------------------------------------------------------
// lse and loss of a row from its (maximum, sum) pairs, joined in a fixed order.  One workgroup takes ROWS rows, 256 / ROWS
// slices of the class tiles each, four pairs in flight per thread: with few rows every row gets a workgroup of its own
// (500 class tiles, one row: 9.8 us with 16 rows per workgroup).
template <int ROWS>
__global__ __launch_bounds__(256) void vh_join(const float2* __restrict__ part, long ldpart, int tiles, const float* __restrict__ zlab,
                                               const int* __restrict__ labels, int n, int classes, int ignore,
                                               float* __restrict__ loss, float* __restrict__ lse) {
  constexpr int SL = 256 / ROWS;
  __shared__ MaxSum red[SL][ROWS];
  const int rl = threadIdx.x % ROWS, sl = threadIdx.x / ROWS, row = blockIdx.x * ROWS + rl;
  MaxSum a = {-INFINITY, 0.f};
  if (row < n) {
    const float2* p = part + row;
    int t = sl;
    for (; t + 3 * SL < tiles; t += 4 * SL) {
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = p[(long)(t + u * SL) * ldpart];
#pragma unroll
      for (int u = 0; u < 4; ++u) a = join(a, {v[u].x, v[u].y});
    }
    for (; t < tiles; t += SL) {
      const float2 v = p[(long)t * ldpart];
      a = join(a, {v.x, v.y});
    }
  }
  red[sl][rl] = a;
  __syncthreads();
#pragma unroll
  for (int w = SL / 2; w > 0; w >>= 1) {
    if (sl < w) red[sl][rl] = join(red[sl][rl], red[sl + w][rl]);
    __syncthreads();
  }
  if (sl || row >= n) return;
  a = red[0][rl];
  // In 64 bits: a loss near zero is the difference of two large numbers.  The exponent of the sum apart, so that the hardware's
  // logarithm (base 2, of 1/2 to 1) is off by a step of 1 at most; divided by the float that the logits were multiplied with.
  const double l = ((double)a.m + (__builtin_amdgcn_frexp_expf(a.s) + (double)__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(a.s)))) /
                   (double)kLog2e;
  lse[row] = (float)l;
  const int y = labels[row];
  loss[row] = y == ignore ? 0.f : (y >= 0 && y < classes ? (float)(l - (double)zlab[row]) : __builtin_nanf(""));
}

// db[v] = scale * sum of the row tiles' partial sums, in order
__global__ __launch_bounds__(256) void vh_dbias(const float* __restrict__ part, long ld, int tiles, float* __restrict__ db, int n,
                                                float scale) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= n) return;
  float s = 0.f;
  for (int t = 0; t < tiles; ++t) s += part[(long)t * ld + v];
  db[v] = s * scale;
}

template <typename T>
__global__ __launch_bounds__(256) void vh_copy(VhCopy c) {
  vh_copy_rows<T>(c, (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256);
}

// out[i] = scale * sum of the slabs, in order, eight loads in flight
template <typename O>
__global__ __launch_bounds__(256) void vh_sum(const float* __restrict__ part, long n, int splits, O* __restrict__ out, float scale) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i + 4 <= n) {
    const float* p = part + i;
    f32x4 s = *reinterpret_cast<const f32x4_any*>(p);
    int k = 1;
    for (; k + 8 <= splits; k += 8) {
      f32x4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const f32x4_any*>(p + (k + u) * n);
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
#pragma unroll 4
    for (; k < splits; ++k) s += *reinterpret_cast<const f32x4_any*>(p + k * n);
    typedef __attribute__((ext_vector_type(4))) O O4;
    s *= scale;
    *reinterpret_cast<O4*>(out + i) = (O4){(O)s[0], (O)s[1], (O)s[2], (O)s[3]};
  } else {
    for (long j = i; j < n; ++j) {
      float s = part[j];
      for (int k = 1; k < splits; ++k) s += part[k * n + j];
      out[j] = (O)(s * scale);
    }
  }
}

}  // namespace dtf

using namespace dtf;

namespace {

constexpr long up(long a, long b) { return (a + b - 1) / b * b; }
constexpr int cdiv(long a, long b) { return (int)((a + b - 1) / b); }
constexpr long kMaxRow = 1L << 20;    // longest row of an operand: a tile's rows are addressed with 32-bit byte offsets
constexpr int kPiece = 256;           // pieces are multiples of this many classes

// Tile configurations, chosen by the number of rows.
//   kSmall: up to 64 rows -- every product streams the weight or its gradient once and is bound by memory: small tiles of the
//           classes / hidden units, several workgroups per CU.
//   kMid:   up to 128 rows: 128 x 64 tiles of four waves, three workgroups per CU (fp32 logits in 64 x 64: 128 rows, 2048 x
//           8000: 73 and 55 us).
//   kLarge: 256 x 256 tiles of eight waves, one workgroup per CU -- or 128 x 128 tiles of four, two per CU, where the large
//           ones leave CUs idle.
enum { kSmall, kMid, kLarge };
int config_for(long n) { return n <= 64 ? kSmall : (n <= 128 ? kMid : kLarge); }

// Tiles of the gradient products
struct GradTile {
  int bm, bn;             // hidden units; rows (dh) or classes (dw)
  int want;               // workgroups that fill the card
};
constexpr GradTile kTiles256{256, 256, 256}, kTiles128{128, 128, 512}, kTiles64{128, 64, 768};
// dh is cut along the classes into as many slabs as it takes to fill the card, so what many large tiles save in operand reads
// few of them lose in slabs: 16 tiles (1000 rows, 1000 x 10007) 42 us against 33 with the small ones, 24 (1500 rows) 55 and 45,
// 32 (4000 rows, 512 x 30000) 139 and 160, 64 (777 rows, 4096 x 50001) 342 and 364.
// fp32 products take a wave all its registers in large tiles, and wait less for each other in small ones (4096 x 1024 x 16000: dh
// 906 and 753 us, dw 931 and 740).
GradTile dh_tile(int E, int cfg, long n, int H) {
  if (cfg != kLarge) return kTiles64;
  return E == 4 || (long)cdiv(H, 256) * cdiv(n, 256) < 32 ? kTiles128 : kTiles256;
}
// dw has its classes to fill the card: rounds over it times their length, 0.57 of a large tile's for two small ones per CU.
// 316 large tiles are two rounds (700 rows, 1024 x 20000: 47 us, small ones 40), 252 are one (500 rows, 1000 x 16000: 23 and 26).
GradTile dw_tile(int E, int cfg, int H, int classes) {
  if (cfg != kLarge) return kTiles64;
  const long large = (long)cdiv(H, 256) * cdiv(classes, 256), small = (long)cdiv(H, 128) * cdiv(classes, 128);
  return E == 4 || 0.57 * cdiv(small, 512) < cdiv(large, 256) ? kTiles128 : kTiles256;
}

// How the logits product of some classes is tiled: the classes below `first` in tiles of one kind, the others in a second one.
// The large kinds run one workgroup per CU, so what counts is the number of rounds over the 256 CUs times the length of a round
// (measured at H = 4096, against 256 x 256, and used at every width: 0.82 for 192 x 256, 0.68 for 256 x 128), and a last round
// for a few tiles is as long as any other: its classes go to small tiles instead.  777 rows x 50001 classes: 784 tiles are four
// rounds, 362 us; three rounds and 91 small tiles 330 us.  Logits of few tiles are cut as small as the CUs hold them at once, because a workgroup alone on its CU takes long over its K (300 rows, 2048 x 5000 bf16: 30 us in large
// tiles, 20 in 200 of 128 x 64; 526 rows, 2944 x 537 fp32: 101 us in 45 tiles of 128 x 64, 52 in 153 of 64 x 32).  Room for
// 512 tiles in bf16 (500 rows, 1000 x 12000: 24 us large, 30 in 752 small ones), 768 in fp32, whose tiles take longer (600 rows,
// 2048 x 8000: 180 us large, 170 in 630 small ones).
struct LogitsTile {
  int bm, bn;
};
struct LogitsTiling {
  LogitsTile kind[2];
  int first;              // classes of the first kind (a multiple of its bm, or all)
  int tiles[2];           // class tiles of either
};
LogitsTiling logits_tiling(int E, int cfg, long n, int classes) {
  LogitsTiling q{{{128, 64}, {128, 64}}, classes, {0, 0}};
  if (cfg == kSmall || (E == 4 && cfg == kMid)) q.kind[0] = {64, E == 4 && n <= 32 ? 32 : 64};
  // the smallest tiles that all CUs hold at once
  const long room = E == 4 ? 768 : 512;
  bool few = false;
  for (const LogitsTile& t : {LogitsTile{32, 32}, LogitsTile{64, 32}, LogitsTile{64, 64}, LogitsTile{128, 64}}) {
    if (few || (E == 2 && (t.bn == 32 || cfg == kSmall)) || (t.bm == 128 && cfg != kLarge)) continue;
    few = (long)cdiv(classes, t.bm) * cdiv(n, t.bn) <= room;
    if (few) q.kind[0] = t;
  }
  if (cfg == kLarge && !few) {
    const struct { LogitsTile t; double length; } kinds[3] = {{{256, 256}, 1.0}, {{192, 256}, 0.82}, {{256, 128}, 0.68}};
    // small tiles: three to a CU; the first of a CU costs more than the next two
    auto small = [&](int rest) {
      const long t = (long)cdiv(rest, 128) * cdiv(n, 64);
      return rest ? 0.16 + 0.14 * cdiv(t, 256) : 0.0;
    };
    double least = 1e30;
    for (const auto& k : kinds) {
      const int rows = cdiv(n, k.t.bn), cols = cdiv(classes, k.t.bm);
      const int full = (int)((long)rows * cols / 256);
      const int some = (int)(full * 256L / rows);          // class tiles that fill whole rounds
      const double whole = cdiv((long)rows * cols, 256) * k.length, split = full * k.length + small(classes - some * k.t.bm);
      if (whole < least) {
        least = whole;
        q.kind[0] = k.t;
        q.first = classes;
      }
      if (some > 0 && some < cols && split < least) {
        least = split;
        q.kind[0] = k.t;
        q.first = some * k.t.bm;
      }
    }
  }
  q.tiles[0] = cdiv(q.first, q.kind[0].bm);
  q.tiles[1] = cdiv(classes - q.first, q.kind[1].bm);
  return q;
}

template <typename T, int BM, int BN, int NWM, int NWN, bool AS, bool BS, int D, class Epi>
int launch(VhOperands p, int splits, const Epi& e, hipStream_t s) {
  p.tiles_m = cdiv(p.M, BM);
  p.tiles_n = cdiv(p.N, BN);
  p.ktiles = cdiv(p.Ka > p.Kb ? p.Ka : p.Kb, 128 / sizeof(T));
  p.splits = splits;
  long grid = (long)p.tiles_m * p.tiles_n * splits;
  if constexpr (Epi::kCopies) grid += e.copy.blocks;
  if (grid > 0x7fffffff) return -1;
  hipLaunchKernelGGL((vh_gemm<T, BM, BN, NWM, NWN, AS, BS, D, Epi>), dim3((unsigned)grid), dim3(NWM * NWN * 64), 0, s, p, e);
  return (int)hipGetLastError();
}

// logits^T [classes][rows] = w . h^T with one kind of tiles
template <typename T, class Epi>
int logits(LogitsTile t, const VhOperands& p, const Epi& e, hipStream_t s) {
  // buffers: 16 rows, 4096 x 32000 bf16: 65.5 us with two, 63.3 with three, 56.1 with four; 128 x 64 tiles of bf16 alone on their
  // CUs gain from a third (prompt of 777 rows: 357 -> 344 us), fp32 ones are long enough
  // fp32: the fewer fragments of the rows' side a wave splits the better (one row, 1024 x 32000: 59 us with 64 rows' tiles of waves
  // side by side, 39 with 32 rows' ones; 64 rows, 1024 x 20000: 56 us side by side, 49 two by two)
  if constexpr (sizeof(T) == 4) {
    if (t.bm == 32) return launch<T, 32, 32, 2, 2, false, false, 4>(p, 1, e, s);
    if (t.bn == 32) return launch<T, 64, 32, 4, 1, false, false, 4>(p, 1, e, s);
    if (t.bm == 64) return launch<T, 64, 64, 2, 2, false, false, 3>(p, 1, e, s);
  } else {
    if (t.bm == 64) return launch<T, 64, 64, 4, 1, false, false, 4>(p, 1, e, s);
  }
  if (t.bm == 128) return launch<T, 128, 64, 2, 2, false, false, sizeof(T) == 2 ? 3 : 2>(p, 1, e, s);
  if (t.bm == 192) return launch<T, 192, 256, 2, 4, false, false, 2>(p, 1, e, s);
  if (t.bn == 128) return launch<T, 256, 128, 4, 2, false, false, 3>(p, 1, e, s);
  return launch<T, 256, 256, 2, 4, false, false, 2>(p, 1, e, s);
}
// The same for all classes: e(kind, first class, first class tile) is the epilogue of a part
template <typename T, class Make>
int logits_all(const LogitsTiling& q, VhOperands p, const Make& make, hipStream_t s) {
  const int classes = p.M;
  for (int k = 0; k < 2; ++k) {
    const int c0 = k ? q.first : 0;
    p.M = k ? classes - q.first : q.first;
    if (!p.M) continue;
    const int rc = logits<T>(q.kind[k], p, make(k, c0, k ? q.tiles[0] : 0), s);
    if (rc) return rc;
    p.A = (const T*)p.A + (long)p.M * p.lda;
  }
  return 0;
}
// dh^T [hidden][rows] = w^T . d^T: the hidden units' side is slow
template <typename T>
int product_dh(int cfg, const GradTile& t, const VhOperands& p, int splits, const VhStore& e, hipStream_t s) {
  if (cfg == kSmall) return launch<T, 128, 64, 4, 1, true, false, 3>(p, splits, e, s);
  if constexpr (sizeof(T) == 2)
    if (t.bn == 256) return launch<T, 256, 256, 2, 4, true, false, 2>(p, splits, e, s);
  if (t.bn == 128) return launch<T, 128, 128, 2, 2, true, false, 2>(p, splits, e, s);
  return launch<T, 128, 64, 2, 2, true, false, 2>(p, splits, e, s);
}
// dw^T [hidden][classes] = h^T . d: both sides slow
template <typename T, bool ONCE>
int product_dw(const GradTile& t, const VhOperands& p, int splits, const VhStoreT<ONCE>& e, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (t.bn == 256) return launch<T, 256, 256, 2, 4, true, true, 2>(p, splits, e, s);
  if (t.bn == 128) return launch<T, 128, 128, 2, 2, true, true, 2>(p, splits, e, s);
  return launch<T, 128, 64, 2, 2, true, true, 2>(p, splits, e, s);
}

// Workgroups that share a tile's K range: where the tiles alone leave CUs idle, the range is cut so that about `want`
// workgroups run, each with at least eight K tiles; their fp32 results are added by vh_sum.
int splits_for(long tiles, int ktiles, int want) {
  long s = want / (tiles < 1 ? 1 : tiles);
  if (s > ktiles / 8) s = ktiles / 8;
  if (s > 64) s = 64;
  if (s < 2) return 1;
  const int per = cdiv(ktiles, s);      // no split without a K tile
  return cdiv(ktiles, per);
}

// Layout of one call's workspace (bytes).  Everything a call needs besides its inputs and outputs.
struct Plan {
  long h_copy, w_copy;      // aligned copies of h (backward: ignored rows zero) and of a piece of w; 0: used as they are
  long part, zlab;          // forward
  long d, sum_h, sum_w, dbpart;
  long total;
  long ldk, ldv;            // padded hidden units, classes of a piece
  int cfg, piece, pieces, splits_h, splits_w;
  int few;                  // d has 64 rows, its rounding errors from row 32 on
  int keep;                 // d has 2 n rows, its rounding errors from row n on
  int drows, rest;          // rows of d; from a row to that of its rounding errors (0: not kept)
  GradTile tile_h, tile_w;
};

int esize(int dtype) { return dtype == 1 ? 2 : 4; }

// Classes per piece: d takes piece * n values.  2^27 of them (256 MB in bf16) leave few, long pieces -- every piece reads and
// writes the fp32 sum of dh once.
int piece_for(long n, int classes) {
  long v = (1L << 27) / (n < 1 ? 1 : n) / kPiece * kPiece;
  if (v < 4 * kPiece) v = 4 * kPiece;
  if (v > kMaxRow) v = kMaxRow;
  return v >= classes ? classes : (int)v;
}

// backward: 1, or 2 with the rounding errors of d kept for any number of rows
Plan plan_for(int dtype, int backward, long n, int H, int V, bool h_ok, bool w_ok, bool bias, int piece) {
  Plan q{};
  const int E = esize(dtype);
  long at = 0;
  auto take = [&](long bytes) {
    const long o = at;
    at += up(bytes, 256);
    return o + 1;           // 0 stands for "none"
  };
  q.cfg = config_for(n);
  q.ldk = up(H, 16 / E);
  q.few = backward && E == 2 && n <= 32;
  q.keep = backward == 2 && E == 2 && !q.few;
  q.rest = q.few ? 32 : (q.keep ? (int)n : 0);
  q.drows = q.few ? 64 : (int)(n + q.rest);
  const long dn = q.drows;
  if (!h_ok || backward) q.h_copy = take(dn * q.ldk * E);
  q.piece = backward ? (piece > 0 ? (int)up(piece, kPiece) : piece_for(n + (q.keep ? n : 0), V)) : V;
  if (q.piece > V) q.piece = V;
  q.pieces = cdiv(V, q.piece);
  if (!w_ok) q.w_copy = take((long)q.piece * q.ldk * E);
  if (!backward) {
    const LogitsTiling t = logits_tiling(E, q.cfg, n, V);
    q.part = take((long)(t.tiles[0] + t.tiles[1]) * n * 8);
    q.zlab = take(n * 4);
  } else {
    const int KT = 128 / E;
    q.ldv = up(q.piece, KT);
    q.d = take(dn * q.ldv * E);
    q.tile_h = dh_tile(E, q.cfg, n, H);
    q.tile_w = dw_tile(E, q.cfg, H, q.piece);
    q.splits_h = splits_for((long)cdiv(H, q.tile_h.bm) * cdiv(q.few ? dn : n, q.tile_h.bn), cdiv(q.ldv, KT), q.tile_h.want);
    q.splits_w = splits_for((long)cdiv(H, q.tile_w.bm) * cdiv(q.piece, q.tile_w.bn), cdiv(dn, KT), q.tile_w.want);
    if (q.pieces > 1 || q.splits_h > 1 || q.keep) q.sum_h = take(q.splits_h * n * H * 4);
    if (q.splits_w > 1) q.sum_w = take(q.splits_w * (long)q.piece * H * 4);
    if (bias) q.dbpart = take((long)cdiv(n, 32) * q.ldv * 4);      // at most that many row tiles
  }
  q.total = at ? at : 256;
  return q;
}

template <typename T>
T* at(void* ws, long o) { return (T*)((char*)ws + o - 1); }

bool rows_ok(const void* p, long ld, int H, int E) { return !((uintptr_t)p & 15) && !(ld * E & 15) && !((long)H * E & 15); }
// The weight is read where it lies if its rows start on 4 bytes and what follows a row of broken 16 bytes is the next row.  (16
// rows, 4095 x 32000 fp32: copied first 332 us forward and 596 backward, read where it lies 116 and 399.)
bool w_rows_ok(const void* p, long ld, int H, int E) {
  return !((uintptr_t)p & 3) && !(ld * E & 3) && (!((long)H * E & 15) || ld == H);
}

template <typename T>
int launch_copy(const VhCopy& c, hipStream_t s) {
  const long chunks = (long)c.R * (c.ldd * (long)sizeof(T) / 16);
  const int grid = chunks > 16384L * 256 ? 16384 : cdiv(chunks, 256);
  hipLaunchKernelGGL(vh_copy<T>, dim3(grid), dim3(256), 0, s, c);
  return (int)hipGetLastError();
}
template <typename O>
int launch_sum(const float* part, long n, int splits, O* out, float scale, hipStream_t s) {
  hipLaunchKernelGGL(vh_sum<O>, dim3(cdiv(n, 1024)), dim3(256), 0, s, part, n, splits, out, scale);
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
  const bool h_ok = rows_ok(h, ldh, H, E), w_ok = w_rows_ok(w, ldw, H, E);
  const Plan q = plan_for(E == 2 ? 1 : 0, 0, n, H, V, h_ok, w_ok, bias != nullptr, 0);
  VhOperands p{w, h, ldw, ldh, V, n, H, (int)q.ldk, 0, 0, 0, 0};
  if (!h_ok) {
    VH_TRY(launch_copy<T>(VhCopy{h, ldh, n, n, H, at<T>(ws, q.h_copy), q.ldk, nullptr, 0, 0, 0}, s));
    p.B = at<T>(ws, q.h_copy);
    p.ldb = q.ldk;
  }
  if (!w_ok) {
    VH_TRY(launch_copy<T>(VhCopy{w, ldw, V, V, H, at<T>(ws, q.w_copy), q.ldk, nullptr, 0, 0, 0}, s));
    p.A = at<T>(ws, q.w_copy);
    p.lda = q.ldk;
    p.Ka = (int)q.ldk;
  }
  const LogitsTiling t = logits_tiling(E, q.cfg, n, V);
  VH_TRY(logits_all<T>(t, p, [&](int, int c0, int tile0) {
    return VhForward{bias ? bias + c0 : nullptr, labels, c0, at<float2>(ws, q.part) + (long)tile0 * n, at<float>(ws, q.zlab), n};
  }, s));
  const int per = n >= 2048 ? 16 : 1;
  hipLaunchKernelGGL((per == 16 ? vh_join<16> : vh_join<1>), dim3(cdiv(n, per)), dim3(256), 0, s, at<float2>(ws, q.part), (long)n,
                     t.tiles[0] + t.tiles[1], at<float>(ws, q.zlab), labels, n, V, ignore, (float*)loss, (float*)lse);
  return (int)hipGetLastError();
}

template <typename T>
int backward(const void* h, long ldh, const void* w, long ldw, const float* bias, const int* labels, const float* lse,
             const float* row_scale, float grad_scale, int n, int H, int V, int ignore, int piece, int keep, void* dh, void* dw,
             int dw_f32, void* db, void* ws, hipStream_t s) {
  const int E = sizeof(T), KT = 128 / E;
  const bool h_ok = rows_ok(h, ldh, H, E);
  const Plan q = plan_for(E == 2 ? 1 : 0, keep ? 2 : 1, n, H, V, h_ok, w_rows_ok(w, ldw, H, E), db != nullptr, piece);
  const T* hp = at<T>(ws, q.h_copy);
  const int dn = q.drows;
  VhCopy copy{h, ldh, q.few ? 32 : n, n, H, at<T>(ws, q.h_copy), q.ldk, labels, ignore, q.rest * q.ldk, 0};
  // Only dw needs the copy where h is aligned: few rows are copied next to the first product (16 rows, 4096 x 32000: 4.5 us less);
  // among large tiles, which hold a CU each, the copy is a launch of its own.
  const bool beside = h_ok && q.cfg != kLarge;
  if (beside) copy.blocks = (int)(copy.R * (q.ldk * E / 16) / 1024 + 1);
  else VH_TRY(launch_copy<T>(copy, s));
  const T* hl = beside ? (const T*)h : hp;
  const long ldl = beside ? ldh : q.ldk;
  for (int k = 0; k < q.pieces; ++k) {
    const int v0 = k * q.piece, vn = V - v0 < q.piece ? V - v0 : q.piece;
    const long ldv = up(vn, KT);
    const T* wp = (const T*)w + (long)v0 * ldw;
    long ldwp = ldw;
    if (q.w_copy) {
      VH_TRY(launch_copy<T>(VhCopy{wp, ldw, vn, vn, H, at<T>(ws, q.w_copy), q.ldk, nullptr, 0, 0, 0}, s));
      wp = at<T>(ws, q.w_copy);
      ldwp = q.ldk;
    }
    T* d = at<T>(ws, q.d);
    const LogitsTiling t = logits_tiling(E, q.cfg, n, vn);
    const VhOperands z{wp, hl, ldwp, ldl, vn, n, q.w_copy ? (int)q.ldk : H, (int)q.ldk, 0, 0, 0, 0};
    auto logits_with = [&](auto keep_d) {
      return logits_all<T>(t, z, [&](int part, int c0, int) {
        VhCopy now = copy;
        if (k || part) now.blocks = 0;
        // one tile of rows: its sums are the whole ones
        const bool whole = n <= t.kind[part].bn;
        float* dbp = !db ? nullptr : whole ? (float*)db + v0 + c0 : at<float>(ws, q.dbpart) + c0;
        return VhGradLogitsT<decltype(keep_d)::value>{
            now, bias ? bias + v0 + c0 : nullptr, labels, lse, row_scale, v0 + c0, V, ignore, d + c0, ldv, q.rest * ldv, (int)ldv - c0, dbp,
            whole ? (part ? vn - t.first : t.first) : (int)ldv - c0, whole ? grad_scale : 1.f};
      }, s);
    };
    if constexpr (sizeof(T) == 2) VH_TRY(q.keep ? logits_with(std::true_type{}) : logits_with(std::false_type{}));
    else VH_TRY(logits_with(std::false_type{}));
    for (int part = 0; db && part < 2; ++part) {
      const int c0 = part ? t.first : 0, cn = part ? vn - t.first : t.first;
      if (!cn || n <= t.kind[part].bn) continue;
      hipLaunchKernelGGL(vh_dbias, dim3(cdiv(cn, 256)), dim3(256), 0, s, at<float>(ws, q.dbpart) + c0, ldv, cdiv(n, t.kind[part].bn),
                         (float*)db + v0 + c0, cn, grad_scale);
      VH_TRY((int)hipGetLastError());
    }
    if (dw) {
      void* out = (char*)dw + (long)v0 * H * (dw_f32 ? 4 : E);
      const bool split = q.splits_w > 1;
      // A large dw would only push other things out of the 256 MB cache (16 rows, 4096 x 32000: 90 us with plain stores, 62 with
      // non-temporal ones); a small one stays for whoever reads it next.
      const bool once = !split && (long)V * H * (dw_f32 ? 4 : E) >= (64L << 20);
      const VhOperands o{hp, d, q.ldk, ldv, H, (int)ldv, dn, dn, 0, 0, 0, 0};
      float* sum = split ? at<float>(ws, q.sum_w) : nullptr;
      if (once) VH_TRY((product_dw<T>(q.tile_w, o, 1, VhStoreT<true>{out, H, dw_f32, 1, vn, sum, 1, 1, grad_scale, 0}, s)));
      else VH_TRY((product_dw<T>(q.tile_w, o, q.splits_w, VhStore{out, H, dw_f32, 1, vn, sum, 1, !split, grad_scale, 0}, s)));
      if (split)
        VH_TRY(dw_f32 ? launch_sum(at<float>(ws, q.sum_w), (long)vn * H, q.splits_w, (float*)out, grad_scale, s)
                      : launch_sum(at<float>(ws, q.sum_w), (long)vn * H, q.splits_w, (T*)out, grad_scale, s));
    }
    if (dh) {
      const bool last = k == q.pieces - 1, split = q.splits_h > 1;
      VhStore st{dh, H, 0, 0, n, q.sum_h ? at<float>(ws, q.sum_h) : nullptr, k == 0, last && !split && !q.keep, grad_scale, q.few};
      VhOperands o{wp, d, ldwp, ldv, H, q.few ? dn : n, vn, (int)ldv, 0, 0, 0, 0};
      VH_TRY((product_dh<T>(q.cfg, q.tile_h, o, q.splits_h, st, s)));
      if (q.keep) {             // the errors' product on top
        o.B = d + q.rest * ldv;
        st.first = 0;
        st.last = last && !split;
        VH_TRY((product_dh<T>(q.cfg, q.tile_h, o, q.splits_h, st, s)));
      }
      if (last && split) VH_TRY(launch_sum(at<float>(ws, q.sum_h), (long)n * H, q.splits_h, (T*)dh, grad_scale, s));
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

// dtype: 0 fp32, 1 bf16.  backward_pass: 1, or 2 for one with keep.  piece: classes per piece of the backward pass (0: the
// default).  Returns < 0 for bad arguments.
long dtf_vocab_head_workspace(int dtype, int backward_pass, const void* h, long ldh, const void* w, long ldw, int n, int H, int V,
                              int bias, int piece) {
  if (!sizes_ok(dtype, n, H, V, ldh, ldw) || backward_pass < 0 || backward_pass > 2 || piece < 0 || piece > kMaxRow) return -3;
  const int E = esize(dtype);
  return plan_for(dtype, backward_pass, n, H, V, rows_ok(h, ldh, H, E), w_rows_ok(w, ldw, H, E), bias != 0, piece).total;
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
// d loss / d loss_i = grad_scale * row_scale[i] (row_scale fp32 [n] or NULL: 1).  keep: bf16 operands keep what rounding drops of d
int dtf_vocab_head_bwd(int dtype, const void* h, long ldh, const void* w, long ldw, const void* bias, const void* labels,
                       const void* lse, const void* row_scale, float grad_scale, int n, int H, int V, int ignore, int piece, int keep,
                       void* dh, void* dw, int dw_f32, void* db, void* ws, long ws_bytes, hipStream_t s) {
  if (!sizes_ok(dtype, n, H, V, ldh, ldw) || !h || !w || !labels || !lse || !ws || ((uintptr_t)ws & 255) || piece < 0 || piece > kMaxRow) return -3;
  if ((uintptr_t)h & (esize(dtype) - 1) || (uintptr_t)w & (esize(dtype) - 1) || ((uintptr_t)dh & 15) || ((uintptr_t)dw & 15)) return -3;
  if (ws_bytes < dtf_vocab_head_workspace(dtype, keep ? 2 : 1, h, ldh, w, ldw, n, H, V, db != nullptr, piece)) return -2;
  return dtype == 1 ? backward<bf16>(h, ldh, w, ldw, (const float*)bias, (const int*)labels, (const float*)lse, (const float*)row_scale,
                                     grad_scale, n, H, V, ignore, piece, keep, dh, dw, dw_f32, db, ws, s)
                    : backward<float>(h, ldh, w, ldw, (const float*)bias, (const int*)labels, (const float*)lse, (const float*)row_scale,
                                      grad_scale, n, H, V, ignore, piece, keep, dh, dw, dw_f32, db, ws, s);
}

}  // extern "C"
