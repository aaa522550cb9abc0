// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft x_0 .. x_{c-1} of a sequence is taken in order while u_i q_i(x_i) < p_i(x_i) (p the target's, q the proposal's
// probability; without a proposal's rows q = 1 on the drafted token).  At the first draft that is refused, i, the token is
// sampled from the remainder (p_i - q_i)+ instead; when all are taken, one more is sampled from p_c.  This leaves the
// target's distribution unchanged.  Sampling inverts the cumulative sum F: the smallest v with F(v) > u F(V - 1).
//
// Whether a token is taken or which v is hit is a comparison at a border, so probabilities are multiplied, subtracted and
// summed in 64 bits: a product of two 32-bit numbers is exact there, and a sum of 2^17 of them is off by 2^-36 at most.
#include "common.h"

typedef _Float16 f16_t;

struct VerifyArgs {
  const int* draft;
  const void *p, *q;
  const float* u;
  const int* counts;
  int *tokens, *accepted;
  long long d_bs, p_bs, p_ns, q_bs, q_ns, u_bs;
  int B, n, V, pad;
};

// How many drafts of sequence b are taken: one lane per draft, the first refusal by ballot.  Every lane gets the answer.
template <typename T>
__device__ __forceinline__ int taken_drafts(const VerifyArgs& a, int b, int lane, int& count) {
  count = a.counts ? max(0, min(a.counts[b], a.n)) : a.n;
  bool ok = false;
  if (lane < count) {
    const int x = a.draft[b * a.d_bs + lane];
    if (x >= 0 && x < a.V) {
      const double pv = (double)(float)((const T*)a.p)[b * a.p_bs + lane * a.p_ns + x];
      const double qv = a.q ? (double)(float)((const T*)a.q)[b * a.q_bs + lane * a.q_ns + x] : 1.0;
      ok = (double)a.u[b * a.u_bs + lane] * qv < pv;
    }
  }
  const unsigned long long refused = ~__ballot(ok);          // n <= 63: lane 63 never takes
  return __ffsll(refused) - 1;
}

struct Rest {          // weights of the row that is sampled from
  const void *p, *q;   // q null: nothing is subtracted, or all of token `gone` (>= 0)
  int gone;
};
template <typename T>
__device__ __forceinline__ double weight(const Rest& r, int v, bool whole) {
  const double pv = (double)(float)((const T*)r.p)[v];
  double w = pv;
  if (!whole) w = r.q ? pv - (double)(float)((const T*)r.q)[v] : (v == r.gone ? pv - 1.0 : pv);
  return w > 0.0 ? w : 0.0;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double wave_scan_f64(double v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  return v;
}

// One workgroup per sequence; wave w sums the w-th contiguous part of the row.
template <typename T>
__global__ __launch_bounds__(1024) void verify_draft_kernel(const VerifyArgs a) {
  __shared__ double s_sum[16];
  __shared__ int s_hit;
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int count;
  const int taken = taken_drafts<T>(a, b, lane, count);
  Rest r{(const T*)a.p + b * a.p_bs + taken * a.p_ns, nullptr, -1};
  if (taken < count) {
    if (a.q) r.q = (const T*)a.q + b * a.q_bs + taken * a.q_ns;
    else r.gone = a.draft[b * a.d_bs + taken];
  }
  const int part = (a.V + 15) / 16, lo = wave * part, hi = min(lo + part, a.V);
  double total = 0.0, before = 0.0, mine = 0.0;
  bool whole = taken >= count;
  for (int tries = 0; tries < 2; ++tries) {
    mine = 0.0;
    for (int v = lo + lane; v < hi; v += 64) mine += weight<T>(r, v, whole);
    mine = wave_sum_f64(mine);
    __syncthreads();
    if (lane == 0) s_sum[wave] = mine;
    if (threadIdx.x == 0) s_hit = 0x7fffffff;
    __syncthreads();
    total = before = 0.0;
    for (int w = 0; w < 16; ++w) {
      if (w == wave) before = total;
      total += s_sum[w];
    }
    if (whole || total > 0.0) break;
    whole = true;                                            // nothing remains: the target's row as it is
  }
  const double u = fmin(fmax((double)a.u[b * a.u_bs + a.n], 0.0), 1.0);
  const double x = u * total;
  if (total > 0.0 && total < INFINITY) {
    // the part that holds the border, or the last part with any weight (u = 1)
    if ((before <= x && before + mine > x) || (x >= total && mine > 0.0 && before + mine == total)) {
      double run = before;
      int best = -1, last = -1;
      for (int v0 = lo; v0 < hi && best < 0; v0 += 64) {
        const int v = v0 + lane;
        const double w = v < hi ? weight<T>(r, v, whole) : 0.0;
        const double f = run + wave_scan_f64(w, lane);
        const unsigned long long hit = __ballot(w > 0.0 && f > x), any = __ballot(w > 0.0);
        if (hit) best = v0 + __ffsll(hit) - 1;
        if (any) last = v0 + 63 - __clzll(any);
        run = __shfl(f, 63, 64);
      }
      if (lane == 0 && (best >= 0 ? best : last) >= 0) atomicMin(&s_hit, best >= 0 ? best : 0x40000000 + last);
    }
  } else if (threadIdx.x == 0) {
    s_hit = 0;                                               // a row without any weight
  }
  __syncthreads();
  if (threadIdx.x <= a.n) {
    int hit = s_hit;
    if (hit >= 0x40000000) hit -= 0x40000000;
    const int j = threadIdx.x;
    a.tokens[(long long)b * (a.n + 1) + j] = j < taken ? a.draft[b * a.d_bs + j] : j == taken ? hit : a.pad;
    if (j == 0) a.accepted[b] = taken;
  }
}

// draft: [B, n] int32, p: [B, n + 1, V], q: [B, n, V] or null, u: [B, n + 1] fp32, counts: [B] or null;
// tokens: [B, n + 1], accepted: [B].  dtype: 0 bf16, 1 fp16, 2 fp32.
extern "C" int dlamd_verify_draft(const void* draft, long long d_bs, const void* p, long long p_bs, long long p_ns,
                                  const void* q, long long q_bs, long long q_ns, const void* u, long long u_bs,
                                  const void* counts, void* tokens, void* accepted, int B, int n, int V, int pad,
                                  int dtype, hipStream_t stream) {
  if (B <= 0) return 0;
  if (n < 0 || n > 63 || V <= 0 || V >= 0x40000000) return -1;
  VerifyArgs a{(const int*)draft, p, q, (const float*)u, (const int*)counts, (int*)tokens, (int*)accepted, d_bs, p_bs, p_ns,
               q_bs, q_ns, u_bs, B, n, V, pad};
  if (dtype == 0) hipLaunchKernelGGL(verify_draft_kernel<bf16_t>, dim3(B), dim3(1024), 0, stream, a);
  else if (dtype == 1) hipLaunchKernelGGL(verify_draft_kernel<f16_t>, dim3(B), dim3(1024), 0, stream, a);
  else if (dtype == 2) hipLaunchKernelGGL(verify_draft_kernel<float>, dim3(B), dim3(1024), 0, stream, a);
  else return -2;
  return DLAMD_CHECK_LAUNCH();
}
