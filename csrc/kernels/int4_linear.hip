// Linear layers with 4-bit weights: y = act(x W^T + bias (+ res)), W[n][k] = (code[n][k] - zero[n][k / G]) scale[n][k / G].
//
// For the few rows of a decode step the layer is a stream of weights: N K / 2 bytes are read once, and everything else is
// small next to them.  Weights lie in the order in which a wave takes them for 16x16x32 matrix instructions:
//     word[N / 16][K / 128][lane][i]   lane = 16 g + r, i < 4:  row 16 t + r, k = 128 s + 32 i + 8 g + (0 .. 7)
// so a lane's 16-byte load holds its operands of four instructions and a wave's load is 1 KB in one piece.  Inside a word
// code 2 p lies in bits 4 p and code 2 p + 1 in bits 16 + 4 p: (word >> 4 p) & 0x000f000f is a pair in two 16-bit halves.
// Scales and zeros are [K / G][N rounded up to 16].
#include "common.h"

typedef _Float16 f16_t;

struct Int4Args {
  const void* x;
  const uint32_t* w;
  const void* scale;
  const uint8_t* zero;
  const float* bias;
  const void* res;
  void* y;
  long long x_rs, res_rs;
  int M, N, K, G, act;
};

// One wave per output column and four rows of x.
template <typename T, typename S>
__global__ __launch_bounds__(256) void int4_linear_kernel(const Int4Args a) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), m0 = blockIdx.y * 4;
  if (n >= a.N) return;
  const int Ks = (a.K + 127) >> 7, Np = (a.N + 15) & ~15;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int e = lane; e < Ks * 16; e += 64) {
    const int s = e >> 4, g = (e >> 2) & 3, i = e & 3;
    const int k = s * 128 + i * 32 + g * 8;
    if (k >= a.K) continue;
    const uint32_t word = a.w[(((long long)(n >> 4) * Ks + s) * 64 + g * 16 + (n & 15)) * 4 + i];
    const long long at = (long long)(k / a.G) * Np + n;
    const float sc = (float)((const S*)a.scale)[at], z = a.zero ? (float)a.zero[at] : 8.f;
    for (int m = 0; m < 4 && m0 + m < a.M; ++m) {
      const T* xr = (const T*)a.x + (m0 + m) * a.x_rs + k;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += (float)xr[j] * ((float)((word >> (4 * (j >> 1) + 16 * (j & 1))) & 15u) - z);
      acc[m] += sum * sc;
    }
  }
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    float v = wave_reduce_sum(acc[m]);
    if (lane == 0 && m0 + m < a.M) {
      if (a.bias) v += a.bias[n];
      if (a.res) v += (float)((const T*)a.res)[(m0 + m) * a.res_rs + n];
      ((T*)a.y)[(long long)(m0 + m) * a.N + n] = (T)dlamd_act(v, a.act);
    }
  }
}

// x: [M, K] (row stride given), y: [M, N] contiguous.  dtype, sdtype: 0 bf16, 1 fp16.  K % G == 0, G 32, 64 or 128.
extern "C" int dlamd_int4_linear(const void* x, long long x_rs, const void* w, const void* scale, const void* zero,
                                 const void* bias, const void* res, long long res_rs, void* y, int M, int N, int K, int G,
                                 int act, int dtype, int sdtype, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || (G != 32 && G != 64 && G != 128) || K % G != 0) return -1;
  if (x_rs % 8 != 0 || (((uintptr_t)x | (uintptr_t)w) & 15)) return -2;
  if ((dtype != 0 && dtype != 1) || (sdtype != 0 && sdtype != 1)) return -3;
  if (act != ACT_NONE && act != ACT_RELU && act != ACT_GELU) return -4;
  Int4Args a{x, (const uint32_t*)w, scale, (const uint8_t*)zero, (const float*)bias, res, y, x_rs, res_rs, M, N, K, G, act};
  const dim3 grid((N + 3) / 4, (M + 3) / 4);
  if (grid.y > 65535) return -5;
  if (dtype == 0 && sdtype == 0) hipLaunchKernelGGL((int4_linear_kernel<bf16_t, bf16_t>), grid, dim3(256), 0, stream, a);
  if (dtype == 0 && sdtype == 1) hipLaunchKernelGGL((int4_linear_kernel<bf16_t, f16_t>), grid, dim3(256), 0, stream, a);
  if (dtype == 1 && sdtype == 0) hipLaunchKernelGGL((int4_linear_kernel<f16_t, bf16_t>), grid, dim3(256), 0, stream, a);
  if (dtype == 1 && sdtype == 1) hipLaunchKernelGGL((int4_linear_kernel<f16_t, f16_t>), grid, dim3(256), 0, stream, a);
  return DLAMD_CHECK_LAUNCH();
}
