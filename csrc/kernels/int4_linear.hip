// Linear layers with 4-bit weights: y = act(x W^T + bias (+ res)), W[n][k] = (code[n][k] - zero[n][k / G]) scale[n][k / G].
//
// For the few rows of a decode step the layer is a stream of weights: N K / 2 bytes are read once, and everything else is
// small next to them.  Weights lie in the order in which a wave takes them for 16x16x32 matrix instructions:
//     word[N / 16][K / 128][lane][i]   lane = 16 g + r, i < 4:  row 16 t + r, k = 128 s + 32 i + 8 g + (0 .. 7)
// so a lane's 16-byte load holds its operands of four instructions and a wave's load is 1 KB in one piece.  Inside a word
// code 2 p lies in bits 4 p and code 2 p + 1 in bits 16 + 4 p: a shift and a mask give a pair in two 16-bit halves.
// Scales and zeros are [K / G][N rounded up to 16].
//
// A code becomes an operand with a shift and one AND-OR: in the top bits of the mantissa of 16 (bits 3 .. 6 in bf16, 6 .. 9 in
// fp16) it is 16 + c, exactly.  The offset leaves again after each group of G features,
//     sum x (c - z) = sum x (16 + c) - (16 + z) sum x,
// where sum x comes from one more matrix instruction (its other operand is all ones), so scale and zero cost one fused
// multiply-add per group and output, not one per weight.  All sums are fp32; at this offset the difference is as exact as a
// sum of the weights' own products (1 to 3e-7 of a layer's typical output).  In the lowest bits codes would need one shift less
// and stand for 128 + c and 1024 + c: 24 x 8192 x 28672 39.4 instead of 39.9 us, and 1e-6 and 2e-5 off.
//
// An infinity in x would make that difference NaN, and so would bf16 values near the end of their range, whose sums with the
// offset overflow: an output that is no finite number is summed once more without the offset (plain4; 24 x 8192 x 28672 with
// an infinity in a row: 2.4 ms).
//
// The waves of a workgroup share R tiles of 16 outputs and split K between them, 128 features at a time; their sums meet in
// LDS.  The next step's loads are in flight while a step is computed.
//
// 5 x 50265 x 1024: 9.6 us, 2.9 TB/s; 1 x 16384 x 4096: 10.9 us; 24 x 8192 x 28672: 39.9 us, 3.1 TB/s.  There a stream of the
// words alone takes 26 us; fetching x (from L2), the scales and the unpacking, scaling and products cost 4 to 8 us each on top,
// which neither x through LDS for eight waves (40 - 46 us), nor more waves over K (44) or over outputs (41 - 42) hid.
// Farther from a stream of their words: 17 to 64 rows of middle-sized layers (48 x 11008 x 4096 24 us, 24 x 7000 x 2048 in groups
// of 64 11.9), where every wave fetches as many bytes of x as of words or more, and from 33 rows on two workgroups fetch and
// unpack the same words; groups of 32 (1 x 20000 x 8192 36.6 us, in groups of 128 22.6), with as many loads of scales and
// zeros as of words; hundreds of rows (600 x 4096 x 4096 59 us), where a word is unpacked again for each 32.
#include "common.h"
#include "decode_abi.h"

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
  float* part;                                               // [kz][M][N rounded up to 16] sums of the parts of K
  int M, N, K, G, act, kw, kz, z_on;                         // z_on: 1, or 0 where `zero` is one word of eights
};

template <typename T> struct Mat4;
template <> struct Mat4<bf16_t> {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t BITS = 0x41804180u, ONE = 0x3f803f80u;
  static constexpr int AT = 3;                               // bit of 1 in a number from 16 to 32
  static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat4<f16_t> {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t BITS = 0x4c004c00u, ONE = 0x3c003c00u;
  static constexpr int AT = 6;
  static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// What a wave holds of one step: 128 features of R tiles of 16 outputs and CT tiles of 16 rows.
template <int R, int CT, int G>
struct Step {
  u32x4 x[CT][4];
  u32x2 s[R][128 / G];                                       // scales of the lane's four outputs
  uint32_t z[R][128 / G];
};

template <int R>
__device__ __forceinline__ void load_words(u32x4 (&w)[R], const Int4Args& a, int s, int tile0, int tiles, int Ks, int lane) {
#pragma unroll
  for (int i = 0; i < R; ++i)
    w[i] = __builtin_nontemporal_load(
        reinterpret_cast<const u32x4*>(a.w + (((long long)min(tile0 + i, tiles - 1) * Ks + s) * 64 + lane) * 4));
}

typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef const uint8_t __attribute__((address_space(1)))* global_u8;    // said to be global memory: a generic load would wait for LDS too
typedef const uint32_t __attribute__((address_space(1)))* global_u32;

// x rows of the workgroup through a bounds-checked buffer: a lane whose row is not there has an offset outside and gets
// zeros without a memory access and without a branch (a branch around loads would make the compiler wait for all of them).
template <int R, int CT, int G>
__device__ __forceinline__ void load_rest(Step<R, CT, G>& t, const Int4Args& a, global_u8 zero, rsrc_t x, const uint32_t (&xo)[CT], int s, int tile0,
                                          int tiles, int g) {
  const int Np = tiles * 16;
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) t.x[c][i] = __builtin_amdgcn_raw_buffer_load_b128(x, xo[c] + 64 * i, s * 256, 0);
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int q = 0; q < 128 / G; ++q) {
      const long long at = (long long)(s * (128 / G) + q) * Np + min(tile0 + i, tiles - 1) * 16 + 4 * g;
      t.s[i][q] = *reinterpret_cast<const u32x2*>((const char*)a.scale + at * 2);
      t.z[i][q] = *(global_u32)(zero + at * a.z_on);
    }
}

// The last step of a K that is no multiple of 128: features from K on are zeros in x.
template <int R, int CT, int G>
__device__ __forceinline__ void load_rest_tail(Step<R, CT, G>& t, const Int4Args& a, global_u8 zero, rsrc_t x, const uint32_t (&xo)[CT], int s,
                                               int tile0, int tiles, int g) {
  const int Np = tiles * 16, groups = a.K / G;
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.x[c][i] = u32x4{0u, 0u, 0u, 0u};
      if (s * 128 + 32 * i < a.K) t.x[c][i] = __builtin_amdgcn_raw_buffer_load_b128(x, xo[c] + 64 * i, s * 256, 0);
    }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int q = 0; q < 128 / G; ++q) {
      const long long at = (long long)min(s * (128 / G) + q, groups - 1) * Np + min(tile0 + i, tiles - 1) * 16 + 4 * g;
      t.s[i][q] = *reinterpret_cast<const u32x2*>((const char*)a.scale + at * 2);
      t.z[i][q] = *(global_u32)(zero + at * a.z_on);
    }
}

// Codes 2 p and 2 p + 1 of a word as a pair of numbers 16 + code.
template <typename T>
__device__ __forceinline__ uint32_t pair_of(uint32_t w, uint32_t mask, int p) {
  constexpr int AT = Mat4<T>::AT;
  return ((4 * p < AT ? w << (AT - 4 * p) : w >> (4 * p - AT)) & mask) | Mat4<T>::BITS;
}

template <typename T, typename S, int R, int CT, int G>
__device__ __forceinline__ void use_step(f32x4 (&y)[R][CT], const u32x4 (&words)[R], const Step<R, CT, G>& t) {
  typedef typename Mat4<T>::x8 x8;
  constexpr uint32_t ONE = Mat4<T>::ONE;
  uint32_t mask = 0x000f000fu << Mat4<T>::AT;
  asm("" : "+v"(mask));                                      // in a vector register: AND-OR takes one scalar operand only
  const x8 ones = __builtin_bit_cast(x8, u32x4{ONE, ONE, ONE, ONE});
#pragma unroll
  for (int q = 0; q < 128 / G; ++q) {
    f32x4 acc[R][CT], xs[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      xs[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < R; ++i) acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i4 = q * (G / 32); i4 < (q + 1) * (G / 32); ++i4) {
#pragma unroll
      for (int c = 0; c < CT; ++c) xs[c] = Mat4<T>::mul(ones, __builtin_bit_cast(x8, t.x[c][i4]), xs[c]);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const uint32_t w = words[i][i4];
        const u32x4 v = {pair_of<T>(w, mask, 0), pair_of<T>(w, mask, 1), pair_of<T>(w, mask, 2), pair_of<T>(w, mask, 3)};
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[i][c] = Mat4<T>::mul(__builtin_bit_cast(x8, v), __builtin_bit_cast(x8, t.x[c][i4]), acc[i][c]);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t h = j & 1 ? t.s[i][q][j >> 1] >> 16 : t.s[i][q][j >> 1] & 0xffffu;
        const float s = (float)__builtin_bit_cast(S, (uint16_t)h);
        const float z = 16.f + (float)((t.z[i][q] >> (8 * j)) & 0xffu);
#pragma unroll
        for (int c = 0; c < CT; ++c) y[i][c][j] += s * (acc[i][c][j] - z * xs[c][j]);
      }
    __builtin_amdgcn_sched_barrier(0);                       // one group's accumulators at a time
  }
}

// Four consecutive sums as they are if they are finite; the others once more, weight by weight.
template <typename T, typename S>
__device__ __forceinline__ f32x4 plain4(const Int4Args& a, f32x4 v, int m, int n) {
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) odd |= !(fabsf(v[j]) < INFINITY);
  if (!odd) return v;
  const int tiles = (a.N + 15) >> 4, Ks = (a.K + 127) >> 7;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int k = 0; k < a.K; k += 8) {
    const auto x = *reinterpret_cast<const typename Mat4<T>::x8*>((const T*)a.x + m * a.x_rs + k);
    const long long at = (long long)(k / a.G) * (tiles * 16) + n;
    const uint32_t* words = a.w + (((long long)(n >> 4) * Ks + (k >> 7)) * 64 + ((k >> 3) & 3) * 16 + (n & 15)) * 4 + ((k >> 5) & 3);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = words[4 * j];
      const float s = (float)((const S*)a.scale)[at + j], z = a.z_on ? (float)a.zero[at + j] : 8.f;
#pragma unroll
      for (int p = 0; p < 8; ++p) y[j] += (float)x[p] * (s * ((float)((w >> (4 * (p >> 1) + 16 * (p & 1))) & 15u) - z));
    }
    if (y[0] != y[0] && y[1] != y[1] && y[2] != y[2] && y[3] != y[3]) break;       // NaN in x: there is no more to find
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = fabsf(v[j]) < INFINITY ? v[j] : y[j];
  return v;
}

// bias, residual, activation, rounding of four consecutive outputs
template <typename T>
__device__ __forceinline__ void finish4(const Int4Args& a, f32x4 v, int m, int n) {
  T* dst = (T*)a.y + (long long)m * a.N + n;
  const T* rs = (const T*)a.res + m * a.res_rs + n;
  T o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j < a.N) {
      float f = v[j];
      if (a.bias) f += a.bias[n + j];
      if (a.res) f += (float)rs[j];
      o[j] = (T)(a.act == ACT_RELU ? (f < 0.f ? 0.f : f) : dlamd_act(f, a.act));      // NaN stays NaN
    }
  }
  if ((a.N & 3) == 0) {
    *reinterpret_cast<u32x2*>(dst) = *reinterpret_cast<u32x2*>(o);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < a.N) dst[j] = o[j];
  }
}

__device__ const uint32_t k_eights = 0x08080808u;             // the zeros of a layer without zeros

// nw x kw waves: wave w takes the tiles of its w / kw and the steps w % kw, + kw, ... of the workgroup's part of K.
template <typename T, typename S, int R, int CT, int G>
__global__ __launch_bounds__(512) void int4_linear_kernel(const Int4Args a) {
  const global_u8 zero = a.z_on ? (global_u8)a.zero : (global_u8)&k_eights;
  extern __shared__ f32x4 s_y[];                             // [kw][nw R CT][lane]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int tiles = (a.N + 15) >> 4, Ks = (a.K + 127) >> 7;
  const int nw = wave / a.kw, kw = wave - nw * a.kw, NW = (blockDim.x >> 6) / a.kw;
  const int wg0 = blockIdx.x * R * NW, tile0 = wg0 + nw * R, m0 = blockIdx.y * 16 * CT;
  const int per = (Ks + a.kz - 1) / a.kz, s0 = blockIdx.z * per, s1 = min(Ks, s0 + per);
  f32x4 y[R][CT];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < CT; ++c) y[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (tile0 < tiles) {
    const int rows = min(16 * CT, a.M - m0);
    const rsrc_t x = __builtin_amdgcn_make_buffer_rsrc((void*)((const T*)a.x + m0 * a.x_rs), 0, (int)((rows - 1) * a.x_rs + a.K) * 2, 0x00020000);
    uint32_t xo[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) xo[c] = 16 * c + r < rows ? (uint32_t)((16 * c + r) * a.x_rs * 2 + 16 * g) : 0x80000000u;
    u32x4 w0[R], w1[R];
    Step<R, CT, G> t0, t1;
    const int full = min(s1, a.K >> 7);                      // steps [s0, full) have all 128 features
    int s = s0 + kw, left = s < full ? (full - 1 - s) / a.kw + 1 : 0;
    if (left == 1) {
      load_words<R>(w0, a, s, tile0, tiles, Ks, lane);
      load_rest<R, CT, G>(t0, a, zero, x, xo, s, tile0, tiles, g);
      __builtin_amdgcn_sched_barrier(0);
      use_step<T, S>(y, w0, t0);
    } else if (left > 1) {
      // Two steps in registers: one computes, one is in flight.  No load here has a condition: where paths with and without
      // a load meet, the compiler can only wait for everything.
      load_words<R>(w0, a, s, tile0, tiles, Ks, lane);
      load_rest<R, CT, G>(t0, a, zero, x, xo, s, tile0, tiles, g);
      __builtin_amdgcn_sched_barrier(0);
      load_words<R>(w1, a, s + a.kw, tile0, tiles, Ks, lane);
      load_rest<R, CT, G>(t1, a, zero, x, xo, s + a.kw, tile0, tiles, g);
      __builtin_amdgcn_sched_barrier(0);
      for (; left > 3; left -= 2, s += 2 * a.kw) {
        use_step<T, S>(y, w0, t0);
        load_words<R>(w0, a, s + 2 * a.kw, tile0, tiles, Ks, lane);
        load_rest<R, CT, G>(t0, a, zero, x, xo, s + 2 * a.kw, tile0, tiles, g);
        __builtin_amdgcn_sched_barrier(0);
        use_step<T, S>(y, w1, t1);
        load_words<R>(w1, a, s + 3 * a.kw, tile0, tiles, Ks, lane);
        load_rest<R, CT, G>(t1, a, zero, x, xo, s + 3 * a.kw, tile0, tiles, g);
        __builtin_amdgcn_sched_barrier(0);
      }
      use_step<T, S>(y, w0, t0);
      if (left == 3) {
        load_words<R>(w0, a, s + 2 * a.kw, tile0, tiles, Ks, lane);
        load_rest<R, CT, G>(t0, a, zero, x, xo, s + 2 * a.kw, tile0, tiles, g);
        __builtin_amdgcn_sched_barrier(0);
        use_step<T, S>(y, w1, t1);
        use_step<T, S>(y, w0, t0);
      } else {
        use_step<T, S>(y, w1, t1);
      }
    }
    const bool tail = full >= s0 && full < s1 && kw == (full - s0) % a.kw;
    if (tail) {
      load_words<R>(w0, a, full, tile0, tiles, Ks, lane);
      load_rest_tail<R, CT, G>(t0, a, zero, x, xo, full, tile0, tiles, g);
      use_step<T, S>(y, w0, t0);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < CT; ++c) s_y[((kw * NW * R + nw * R + i) * CT + c) * 64 + lane] = y[i][c];
  __syncthreads();
  // an item: four consecutive outputs of one row; consecutive threads take consecutive outputs
  const int RT = R * NW;
  for (int e = threadIdx.x; e < RT * CT * 64; e += blockDim.x) {
    const int q = e % (4 * RT), rest = e / (4 * RT), rr = rest & 15, c = rest >> 4;
    const int i = q >> 2, l = (q & 3) * 16 + rr;
    const int m = m0 + 16 * c + rr, n = (wg0 + i) * 16 + 4 * (q & 3);
    if (m >= a.M || n >= a.N) continue;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < a.kw; ++w) {
      const f32x4 t = s_y[((w * RT + i) * CT + c) * 64 + l];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += t[j];
    }
    if (a.kz == 1) finish4<T>(a, plain4<T, S>(a, v, m, n), m, n);
    else *reinterpret_cast<f32x4*>(a.part + ((long long)blockIdx.z * a.M + m) * (tiles * 16) + n) = v;
  }
}

// Sums the parts of K and finishes: a thread per four outputs.
template <typename T, typename S>
__global__ __launch_bounds__(256) void int4_join_kernel(const Int4Args a) {
  const int Np = (a.N + 15) & ~15, per = Np >> 2;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(e / per), n = (int)(e - (long long)m * per) * 4;
  if (m >= a.M || n >= a.N) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int z = 0; z < a.kz; ++z) {
    const f32x4 t = *reinterpret_cast<const f32x4*>(a.part + ((long long)z * a.M + m) * Np + n);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += t[j];
  }
  finish4<T>(a, plain4<T, S>(a, v, m, n), m, n);
}

template <typename T, typename S, int R, int CT, int G>
static void launch4(const Int4Args& a, int nw, hipStream_t stream) {
  const int per = R * nw;
  const dim3 grid(((a.N + 15) / 16 + per - 1) / per, (a.M + 16 * CT - 1) / (16 * CT), a.kz);
  hipLaunchKernelGGL((int4_linear_kernel<T, S, R, CT, G>), grid, dim3(nw * a.kw * 64), nw * a.kw * R * CT * 1024, stream, a);
  if (a.kz > 1) {
    const long long items = (long long)a.M * ((a.N + 15) / 16 * 4);
    hipLaunchKernelGGL((int4_join_kernel<T, S>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, a);
  }
}
template <typename T, typename S, int R, int CT>
static void launch4_g(const Int4Args& a, int G, int nw, hipStream_t stream) {
  constexpr int R32 = R * CT == 8 ? 2 : R;                   // the scales of groups of 32 and 8 tiles do not fit the registers;
                                                             // of groups of 64 all but 10 to 17 do, which go to scratch
  if (G == 32) launch4<T, S, R32, CT, 32>(a, nw, stream);
  else if (G == 64) launch4<T, S, R, CT, 64>(a, nw, stream);
  else launch4<T, S, R, CT, 128>(a, nw, stream);
}
template <typename T, typename S>
static void launch4_r(const Int4Args& a, int R, int CT, int G, int nw, hipStream_t stream) {
  if (CT == 1) {
    if (R == 1) launch4_g<T, S, 1, 1>(a, G, nw, stream);
    else launch4_g<T, S, 2, 1>(a, G, nw, stream);
  } else {
    if (R == 1) launch4_g<T, S, 1, 2>(a, G, nw, stream);
    else launch4_g<T, S, 4, 2>(a, G, nw, stream);
  }
}

// x: [M, K] (row stride given), y: [M, N] contiguous.  dtype, sdtype: 0 bf16, 1 fp16.  K % G == 0, G 32, 64 or 128.
// A wave holds `tiles` tiles of 16 outputs (1, or 2 up to 16 rows and 4 from there), a workgroup nw x kw <= 8 waves, K is split
// into kz parts over workgroups (part: [kz][M][N rounded up to 16] floats where kz > 1).
extern "C" int dlamd_int4_linear(const void* x, long long x_rs, const void* w, const void* scale, const void* zero,
                                 const void* bias, const void* res, long long res_rs, void* y, int M, int N, int K, int G,
                                 int act, int dtype, int sdtype, int tiles, int nw, int kw, int kz, void* part,
                                 long long part_floats, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || (G != 32 && G != 64 && G != 128) || K % G != 0 || N > 1 << 26) return -1;
  if (x_rs < 0 || x_rs >= (1 << 24) || K >= (1 << 24)) return -9;   // a workgroup's 32 rows of x: 31-bit offsets
  if (x_rs % 8 != 0 || (((uintptr_t)x | (uintptr_t)w) & 15) || ((uintptr_t)scale & 7) || ((uintptr_t)zero & 3) || ((uintptr_t)y & 7)) return -2;
  if ((dtype != 0 && dtype != 1) || (sdtype != 0 && sdtype != 1)) return -3;
  if (act != ACT_NONE && act != ACT_RELU && act != ACT_GELU) return -4;
  const int CT = M <= 16 ? 1 : 2;
  if ((M + 16 * CT - 1) / (16 * CT) > 65535) return -5;
  if ((tiles != 1 && tiles != 2 * CT) || nw < 1 || kw < 1 || nw * kw > 8 || nw * kw * tiles * CT > 64) return -6;
  if (kz < 1 || kz > 64 || (kz > 1 && (!part || ((uintptr_t)part & 15) || part_floats < (long long)kz * M * ((N + 15) / 16 * 16)))) return -7;
  if (kz > 1 && (long long)M * ((N + 15) / 16 * 4) > 0xffffff00LL) return -8;      // a launch has fewer than 2^32 threads
  Int4Args a{x, (const uint32_t*)w, scale, (const uint8_t*)zero, (const float*)bias, res, y, x_rs, res_rs, (float*)part,
             M, N, K, G, act, kw, kz, zero ? 1 : 0};
  if (dtype == 0 && sdtype == 0) launch4_r<bf16_t, bf16_t>(a, tiles, CT, G, nw, stream);
  if (dtype == 0 && sdtype == 1) launch4_r<bf16_t, f16_t>(a, tiles, CT, G, nw, stream);
  if (dtype == 1 && sdtype == 0) launch4_r<f16_t, bf16_t>(a, tiles, CT, G, nw, stream);
  if (dtype == 1 && sdtype == 1) launch4_r<f16_t, f16_t>(a, tiles, CT, G, nw, stream);
  return DLAMD_CHECK_LAUNCH();
}
