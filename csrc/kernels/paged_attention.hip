// Attention of one or a few new tokens per sequence over a paged key / value cache.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the visible positions j of the sequence, one pass over keys and values with
// the running maximum m and sum l of the softmax (a new maximum rescales what is summed so far by exp(m_old - m_new)).
// A position is visible when it is below the sequence's limit and its page exists; keys and values of other positions
// are never used in arithmetic, whatever they hold.  A row without visible positions is 0, its log-sum-exp -inf.
#include "common.h"

typedef _Float16 f16_t;

struct PagedAttArgs {
  const void *q, *kp, *vp;
  void* o;
  float* lse;
  const int *table, *lens;
  long long q_bs, q_ns, q_hs;
  long long kp_ps, kp_ss, kp_hs, vp_ps, vp_ss, vp_hs, t_bs;
  int B, n, Hq, Hkv, page, width, pages, causal;
  float scale;
};

// One wave per query row: 8 dimensions per lane, D / 8 lanes per key, 64 / (D / 8) keys side by side.
template <typename T, int D>
__global__ __launch_bounds__(64) void paged_attention_kernel(const PagedAttArgs p) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  constexpr int LK = D / 8, KEYS = 64 / LK;
  const int row = blockIdx.x;
  const int h = row % p.Hq, i = (row / p.Hq) % p.n, b = row / (p.Hq * p.n);
  const int hk = h / (p.Hq / p.Hkv);
  const int lane = threadIdx.x, sub = lane % LK, kq = lane / LK;
  const int kept = p.lens[b];
  long long limit = kept < 0 ? 0 : (long long)kept + (p.causal ? i + 1 : 0);
  limit = min(limit, (long long)p.width * p.page);
  float qv[8];
  {
    const T8 t = *reinterpret_cast<const T8*>((const T*)p.q + b * p.q_bs + i * p.q_ns + h * p.q_hs + sub * 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) qv[j] = (float)t[j];
  }
  float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (long long k0 = 0; k0 < limit; k0 += KEYS) {
    const long long pos = k0 + kq;
    int pid = pos < limit ? p.table[b * p.t_bs + pos / p.page] : -1;
    const bool ok = pid >= 0 && pid < p.pages;
    const long long slot = pos % p.page;
    float s = 0.f;
    T8 vt;
    if (ok) {
      const T8 kt = *reinterpret_cast<const T8*>((const T*)p.kp + pid * p.kp_ps + slot * p.kp_ss + hk * p.kp_hs + sub * 8);
      vt = *reinterpret_cast<const T8*>((const T*)p.vp + pid * p.vp_ps + slot * p.vp_ss + hk * p.vp_hs + sub * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += qv[j] * (float)kt[j];
    }
#pragma unroll
    for (int x = 1; x < LK; x <<= 1) s += __shfl_xor(s, x, 64);
    if (ok) {
      s *= p.scale;
      const float mn = fmaxf(m, s);
      const float a = m == -INFINITY ? 0.f : __expf(m - mn), e = s == -INFINITY ? 0.f : __expf(s - mn);
      l = l * a + e;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = acc[j] * a + e * (float)vt[j];
      m = mn;
    }
  }
#pragma unroll
  for (int x = LK; x < 64; x <<= 1) {
    const float mo = __shfl_xor(m, x, 64), lo = __shfl_xor(l, x, 64), mn = fmaxf(m, mo);
    const float a = m == -INFINITY ? 0.f : __expf(m - mn), c = mo == -INFINITY ? 0.f : __expf(mo - mn);
    l = l * a + lo * c;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = acc[j] * a + __shfl_xor(acc[j], x, 64) * c;
    m = mn;
  }
  if (kq == 0) {
    T8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (T)(l > 0.f ? acc[j] / l : 0.f);
    *reinterpret_cast<T8*>((T*)p.o + (long long)row * D + sub * 8) = o;
    if (p.lse && sub == 0) p.lse[row] = l > 0.f ? m + __logf(l) : -INFINITY;
  }
}

// q: [B, n, Hq, D] (strides given), o: [B, n, Hq, D] contiguous, lse: [B, n, Hq] or null.  dtype: 0 bf16, 1 fp16.
extern "C" int dlamd_paged_attention(const void* q, long long q_bs, long long q_ns, long long q_hs, const void* kp,
                                     long long kp_ps, long long kp_ss, long long kp_hs, const void* vp, long long vp_ps,
                                     long long vp_ss, long long vp_hs, const void* table, long long t_bs,
                                     const void* lens, void* o, void* lse, int B, int n, int Hq, int Hkv, int D, int page,
                                     int width, int pages, int causal, float scale, int dtype, hipStream_t stream) {
  if (B <= 0 || n <= 0 || Hq <= 0) return 0;
  if (Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128)) return -1;
  if (page <= 0 || page % 16 != 0 || width < 0 || pages < 0) return -2;
  if ((q_bs | q_ns | q_hs | kp_ps | kp_ss | kp_hs | vp_ps | vp_ss | vp_hs) % 8 != 0) return -3;
  if (((uintptr_t)q | (uintptr_t)kp | (uintptr_t)vp | (uintptr_t)o) & 15) return -4;
  if ((long long)B * n * Hq > 0x7fffffffLL) return -5;
  if (dtype != 0 && dtype != 1) return -6;
  PagedAttArgs a{q, kp, vp, o, (float*)lse, (const int*)table, (const int*)lens, q_bs, q_ns, q_hs,
                 kp_ps, kp_ss, kp_hs, vp_ps, vp_ss, vp_hs, t_bs, B, n, Hq, Hkv, page, width, pages, causal, scale};
  const dim3 grid((unsigned)(B * n * Hq));
  if (dtype == 0 && D == 64) hipLaunchKernelGGL((paged_attention_kernel<bf16_t, 64>), grid, dim3(64), 0, stream, a);
  if (dtype == 0 && D == 128) hipLaunchKernelGGL((paged_attention_kernel<bf16_t, 128>), grid, dim3(64), 0, stream, a);
  if (dtype == 1 && D == 64) hipLaunchKernelGGL((paged_attention_kernel<f16_t, 64>), grid, dim3(64), 0, stream, a);
  if (dtype == 1 && D == 128) hipLaunchKernelGGL((paged_attention_kernel<f16_t, 128>), grid, dim3(64), 0, stream, a);
  return DLAMD_CHECK_LAUNCH();
}
