// Pure-MFMA micro-benchmark: what is the MFMA issue rate of this chip under load, and at which clock?
// (in-kernel stamps said 1.785 GHz, rocm-smi 2.35 GHz -- a 30 % uncertainty in every "% of peak".)
// Every wave runs N v_mfma_f32_16x16x32_bf16 back to back, either on ONE accumulator (dependent chain) or on FOUR
// (independent: the pipe's issue rate), stamps s_memtime (shader-clock counter) and s_memrealtime (100 MHz wall clock)
// around the loop, and the host prints cycles per MFMA, ns per MFMA and the clock the two counters imply.
//   hipcc $(python3 tools/build_native.py --flags) -o mfma_rate tools/micro/mfma_rate.hip && ./mfma_rate
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include <algorithm>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

template <int INDEP>
__global__ __launch_bounds__(1024) void mfma_loop(int iters, long long* stamps, float* sink) {
  bf16x8 a, b;
  for (int j = 0; j < 8; ++j) {
    a[j] = (__bf16)(0.001f * (threadIdx.x + j));
    b[j] = (__bf16)(0.002f * (threadIdx.x - j));
  }
  f32x4 acc[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
  __syncthreads();
  const long long c0 = clock64(), w0 = wall_clock64();
  f32x4 acc4 = acc[0], acc5 = acc[0], acc6 = acc[0], acc7 = acc[0];
  // inline asm with explicit accumulators: through the builtin the compiler rotates the four accumulators through
  // overlapping register tuples (a[0:3] <- a[2:5] ...), which adds dependencies of its own to the "independent" loop
#define MFMA(ACC) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(ACC) : "v"(a), "v"(b))
  for (int i = 0; i < iters; ++i) {
    if (INDEP == 1) {
#pragma unroll
      for (int u = 0; u < 16; ++u) MFMA(acc[0]);
    } else {
      MFMA(acc[0]); MFMA(acc[1]); MFMA(acc[2]); MFMA(acc[3]); MFMA(acc4); MFMA(acc5); MFMA(acc6); MFMA(acc7);
      MFMA(acc[0]); MFMA(acc[1]); MFMA(acc[2]); MFMA(acc[3]); MFMA(acc4); MFMA(acc5); MFMA(acc6); MFMA(acc7);
    }
  }
  // the accumulators are read before the second stamp: the MFMAs have completed
  float s = acc[0][0] + acc[1][1] + acc[2][2] + acc[3][3] + acc4[0] + acc5[1] + acc6[2] + acc7[3];
  asm volatile("" : "+v"(s));
  const long long c1 = clock64(), w1 = wall_clock64();
  if ((threadIdx.x & 63) == 0) {
    const size_t wave = (size_t)blockIdx.x * (blockDim.x / 64) + threadIdx.x / 64;
    stamps[2 * wave] = c1 - c0;
    stamps[2 * wave + 1] = w1 - w0;
  }
  if (s == 123.456f) *sink = s;
}

template <int INDEP>
static void run(const char* what, int blocks, int threads, int iters) {
  const int waves = blocks * threads / 64;
  long long* d;
  float* sink;
  hipMalloc(&d, sizeof(long long) * 2 * waves);
  hipMalloc(&sink, 4);
  for (int rep = 0; rep < 3; ++rep) hipLaunchKernelGGL(mfma_loop<INDEP>, dim3(blocks), dim3(threads), 0, 0, iters, d, sink);
  hipDeviceSynchronize();
  std::vector<long long> h(2 * waves);
  hipMemcpy(h.data(), d, sizeof(long long) * 2 * waves, hipMemcpyDeviceToHost);
  std::vector<double> cyc(waves), ns(waves);
  for (int w = 0; w < waves; ++w) {
    cyc[w] = (double)h[2 * w] / (16.0 * iters);
    ns[w] = (double)h[2 * w + 1] * 10.0 / (16.0 * iters);
  }
  std::sort(cyc.begin(), cyc.end());
  std::sort(ns.begin(), ns.end());
  const double c = cyc[waves / 2], n = ns[waves / 2];
  printf("%-58s %5d wg x %3d thr: %6.2f s_memtime ticks / MFMA, %6.2f ns / MFMA (median wave)  -> s_memtime runs at %7.1f MHz\n",
         what, blocks, threads, c, n, c / n * 1e3);
  hipFree(d);
  hipFree(sink);
}

int main() {
  hipDeviceProp_t p;
  hipGetDeviceProperties(&p, 0);
  printf("%s, %d CUs, clockRate %d kHz\n", p.name, p.multiProcessorCount, p.clockRate);
  const int cus = p.multiProcessorCount;
  // 16 x 16 x 32 bf16 = 16384 FLOP.  One wave per SIMD (256 threads per CU) and two (512).
  run<1>("dependent chain, 1 wave / SIMD, every CU", cus, 256, 4096);
  run<4>("8 independent accumulators, 1 wave / SIMD, every CU", cus, 256, 4096);
  run<4>("8 independent accumulators, 2 waves / SIMD, every CU", cus, 512, 4096);
  run<4>("8 independent accumulators, 4 waves / SIMD, every CU", cus, 1024, 4096);
  run<4>("8 independent accumulators, 1 wave / SIMD, ONE CU", 1, 256, 4096);
  run<4>("8 independent accumulators, 1 wave on ONE SIMD", 1, 64, 4096);
  printf("(per SIMD: ns / MFMA with one wave per SIMD; with two waves per SIMD each wave gets every other slot, so the pipe's\n"
         " interval is half the per-wave figure.  FLOP/s of the chip = CUs x 4 SIMDs x 16384 / interval.)\n");
  return 0;
}
