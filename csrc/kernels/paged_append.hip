// Appending keys and values of new tokens to a paged cache, with the position rotation on the way.
//
// Token t is the i-th new token of sequence b; its position is lens[b] + i, its place the slot pos % page of the page
// table[b][pos / page].  The first `rot` dimensions of every key (and query) head turn by the position's angles,
//     (a, b) -> (a cos - b sin, a sin + b cos),
// pairs being (d, d + rot / 2) or, interleaved, (2 d, 2 d + 1); the maths is fp32, rounded once at the store.
//
// Pure data movement (every byte is read once and written once), so the kernel is a flat list of 16-byte units: a unit
// is one 8-dimension chunk, or, for half-split pairs, the two chunks that turn into each other.  A workgroup per token keeps
// the page, the slot and the angles' row uniform.  16384 packed prompt tokens, 32 + 2 x 8 heads of 128: 79.7 us, 5.0 TB/s, what
// a copy reaches; one token each for 16 sequences takes 2.9 us on the device, three dependent fetches.
#include "common.h"
#include "decode_abi.h"

typedef _Float16 f16_t;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct AppendArgs {
  const void *k, *v, *q;
  void *kp, *vp, *qo;
  const int *table, *lens, *starts;
  const float *cs, *sn;
  long long k_ts, k_hs, v_ts, v_hs, q_ts, q_hs;              // token / head strides, elements
  long long kp_ps, kp_ss, kp_hs, vp_ps, vp_ss, vp_hs;        // page / slot / head strides, elements
  long long t_bs;                                            // table row stride
  int B, T, n, Hq, Hkv, D, rot, page, width, pages, interleaved;
};

template <typename T8>
__device__ __forceinline__ void load8(const void* p, long long off, float* f) {
  const T8 t = *reinterpret_cast<const T8*>(reinterpret_cast<const char*>(p) + off * 2);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)t[j];
}
template <typename T8, typename T>
__device__ __forceinline__ void store8(void* p, long long off, const float* f) {
  T8 t;
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = (T)f[j];
  *reinterpret_cast<T8*>(reinterpret_cast<char*>(p) + off * 2) = t;
}

// One workgroup per token.
template <typename T8, typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs p) {
  const int t = blockIdx.x;
  int b, i;
  if (p.starts) {
    // the sequence is the number of sequence ends at or before t: lanes compare, ballots count
    b = 0;
    for (int s0 = 0; s0 < p.B; s0 += 64) {
      const int s = s0 + (threadIdx.x & 63);
      b += __popcll(__ballot(s < p.B && p.starts[s + 1] <= t));
    }
    i = b < p.B ? t - p.starts[b] : -1;
  } else {
    b = t / p.n;
    i = t - b * p.n;
  }
  long long pos = -1;
  int pid = -1;
  if (b < p.B && i >= 0) {
    const int kept = p.lens[b];
    pos = (long long)kept + i;
    if (kept < 0 || pos >= (long long)p.width * p.page) pos = -1;
    if (pos >= 0) {
      pid = p.table[b * p.t_bs + pos / p.page];
      if (pid >= p.pages) pid = -1;
    }
  }
  const int slot = pos >= 0 ? (int)(pos % p.page) : 0;
  const int half = p.rot >> 1;
  const int chunks = p.D >> 3;
  const int pairs = p.interleaved ? 0 : p.rot >> 4;          // units of two chunks per rotated head
  const int per = chunks - pairs;                            // units per rotated head
  const int nq = p.q ? p.Hq * per : 0, nk = p.Hkv * per, nv = p.Hkv * chunks;
  for (int u = threadIdx.x; u < nq + nk + nv; u += 256) {
    if (u >= nq + nk) {
      if (pid < 0) continue;
      const int r = u - nq - nk, h = r / chunks, c = r - h * chunks;
      const long long src = t * p.v_ts + h * p.v_hs + c * 8, dst = pid * p.vp_ps + slot * p.vp_ss + h * p.vp_hs + c * 8;
      *reinterpret_cast<u32x4*>((char*)p.vp + dst * 2) = *reinterpret_cast<const u32x4*>((const char*)p.v + src * 2);
      continue;
    }
    const bool isq = u < nq;
    const int r = isq ? u : u - nq, h = r / per, c = r - h * per;
    if (!isq && pid < 0) continue;
    const void* src = isq ? p.q : p.k;
    void* dst = isq ? p.qo : p.kp;
    const long long so = isq ? t * p.q_ts + h * p.q_hs : t * p.k_ts + h * p.k_hs;
    const long long dn = isq ? ((long long)t * p.Hq + h) * p.D : pid * p.kp_ps + slot * p.kp_ss + h * p.kp_hs;
    const int d = c < pairs ? c * 8 : (c + pairs) * 8;       // first dimension of the unit
    if (isq && pos < 0) {                                    // a query of no sequence
      *reinterpret_cast<u32x4*>((char*)dst + (dn + d) * 2) = u32x4{0u, 0u, 0u, 0u};
      if (c < pairs) *reinterpret_cast<u32x4*>((char*)dst + (dn + d + half) * 2) = u32x4{0u, 0u, 0u, 0u};
      continue;
    }
    float x[8], y[8];
    load8<T8>(src, so + d, x);
    if (c < pairs) {
      load8<T8>(src, so + d + half, y);
      float a[8], e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float cv = p.cs[pos * half + d + j], sv = p.sn[pos * half + d + j];
        a[j] = x[j] * cv - y[j] * sv;
        e[j] = x[j] * sv + y[j] * cv;
      }
      store8<T8, T>(dst, dn + d, a);
      store8<T8, T>(dst, dn + d + half, e);
    } else {
      if (p.interleaved && d < p.rot) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float cv = p.cs[pos * half + (d + j) / 2], sv = p.sn[pos * half + (d + j) / 2];
          const float a = x[j] * cv - x[j + 1] * sv;
          x[j + 1] = x[j] * sv + x[j + 1] * cv;
          x[j] = a;
        }
      }
      store8<T8, T>(dst, dn + d, x);
    }
  }
}

// k, v: [T, Hkv, D] (strides given, last dimension contiguous), q: [T, Hq, D] or null, qo: [T, Hq, D] contiguous.
// kp, vp: [pages, page, Hkv, D].  starts: [B + 1] or null (then n tokens per sequence).  dtype: 0 bf16, 1 fp16.
extern "C" int dlamd_paged_append(const void* k, long long k_ts, long long k_hs, const void* v, long long v_ts,
                                  long long v_hs, const void* q, long long q_ts, long long q_hs, void* qo, void* kp,
                                  long long kp_ps, long long kp_ss, long long kp_hs, void* vp, long long vp_ps,
                                  long long vp_ss, long long vp_hs, const void* table, long long t_bs, const void* lens,
                                  const void* starts, const void* cs, const void* sn, int B, int T, int Hq, int Hkv,
                                  int D, int rot, int page, int width, int pages, int interleaved, int dtype,
                                  hipStream_t stream) {
  if (B <= 0 || T <= 0 || Hkv <= 0 || width <= 0) return 0;
  if (D <= 0 || D % 8 != 0 || page <= 0 || pages < 0) return -1;
  if (rot < 0 || rot > D || rot % 16 != 0 || (rot > 0 && (!cs || !sn))) return -2;
  if ((q != nullptr) != (qo != nullptr) || (q && Hq <= 0)) return -3;
  if (!starts && T % B != 0) return -4;
  if ((k_ts | k_hs | v_ts | v_hs | kp_ps | kp_ss | kp_hs | vp_ps | vp_ss | vp_hs) % 8 != 0 || (q && (q_ts | q_hs) % 8 != 0)) return -5;
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)qo | (uintptr_t)kp | (uintptr_t)vp) & 15) return -6;
  if (dtype != 0 && dtype != 1) return -7;
  if (T >= 1 << 24) return -8;                               // a launch has fewer than 2^32 threads
  AppendArgs a{k, v, q, kp, vp, qo, (const int*)table, (const int*)lens, (const int*)starts, (const float*)cs, (const float*)sn,
               k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, kp_ps, kp_ss, kp_hs, vp_ps, vp_ss, vp_hs, t_bs,
               B, T, starts ? 0 : T / B, Hq, Hkv, D, rot, page, width, pages, interleaved};
  if (dtype == 0)
    hipLaunchKernelGGL((paged_append_kernel<bf16x8, bf16_t>), dim3(T), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_append_kernel<f16x8, f16_t>), dim3(T), dim3(256), 0, stream, a);
  return DLAMD_CHECK_LAUNCH();
}
