// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft x_0 .. x_{c-1} of a sequence is taken in order while u_i q_i(x_i) < p_i(x_i) (p the target's, q the proposal's
// probability; without a proposal's rows q = 1 on the drafted token).  At the first draft that is refused, i, the token is
// sampled from the remainder (p_i - q_i)+ instead; when all are taken, one more is sampled from p_c.  This leaves the
// target's distribution unchanged.  Sampling inverts the cumulative sum F: the smallest v with F(v) > u F(V - 1).
//
// Whether a token is taken or which v is hit is a comparison at a border, so probabilities are multiplied, subtracted and
// summed in 64 bits: a product of two 32-bit numbers is exact there, and a sum of 2^17 of them is off by 2^-36 at most.
//
// Two rows per sequence are read once, the drafted probabilities before them (a gather each), the piece with the border after
// the sums: a chain of dependent fetches, hence rows in registers up to 8192 tokens (8 x 4000: 5.8 us), pieces over several
// workgroups and a second launch beyond (1 x 50265: 9.6 us, 8.0 in a graph, 3.4 + 4.3 on the device; 192 x 50265: 22 us,
// 3.5 TB/s).
#include "common.h"
#include "decode_abi.h"

typedef _Float16 f16_t;

struct VerifyArgs {
  const int* draft;
  const void *p, *q;
  const float* u;
  const int* counts;
  int *tokens, *accepted;
  long long d_bs, p_bs, p_ns, q_bs, q_ns, u_bs;
  double* sums;                                              // [B][pieces]: weight of the rest, of the whole row
  int B, n, V, pad, pieces;
};

// How many drafts of sequence b are taken: one lane per draft, the first refusal by ballot.  Every lane gets the answer.
template <typename T>
__device__ __forceinline__ int taken_drafts(const VerifyArgs& a, int b, int lane) {
  bool ok = false;
  if (lane < a.n) {
    const int count = a.counts ? a.counts[b] : a.n, x = a.draft[b * a.d_bs + lane];
    const float u = a.u[b * a.u_bs + lane];
    if (lane < count && x >= 0 && x < a.V) {
      const T pv = ((const T*)a.p)[b * a.p_bs + lane * a.p_ns + x];
      const double qv = a.q ? (double)(float)((const T*)a.q)[b * a.q_bs + lane * a.q_ns + x] : 1.0;
      ok = (double)u * qv < (double)(float)pv;
    }
  }
  return __ffsll((long long)~__ballot(ok)) - 1;              // n <= 63: lane 63 never takes
}

// The row that is sampled from: weights (p - q)+, or p with the probability of token `gone` less one, or p itself (whole).
template <typename T>
struct Rest {
  const T *p, *q;                                            // q null: only `gone` (if >= 0) loses
  int gone;
  __device__ __forceinline__ Rest(const VerifyArgs& a, int b, int taken) {
    const int count = a.counts ? min(a.counts[b], a.n) : a.n;
    p = (const T*)a.p + b * a.p_bs + taken * a.p_ns;
    q = a.q && taken < count ? (const T*)a.q + b * a.q_bs + taken * a.q_ns : nullptr;
    gone = !a.q && taken < count ? a.draft[b * a.d_bs + taken] : -1;
  }
};
__device__ __forceinline__ double positive(double w) { return w > 0.0 ? w : 0.0; }    // NaN weighs nothing

// Weights of U tokens, `step` apart; none from `end` on.  All loads are in flight at once.
template <typename T, bool Q, int U>
__device__ __forceinline__ void weights_of(const Rest<T>& r, int v, int end, int step, double (&rest)[U], double (&whole)[U]) {
  T p[U], q[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int at = min(v + i * step, end - 1);
    p[i] = r.p[at];
    if (Q) q[i] = r.q[at];
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const bool in = v + i * step < end;
    const double w = (double)(float)p[i];
    whole[i] = in ? positive(w) : 0.0;
    rest[i] = in ? positive(Q ? w - (double)(float)q[i] : v + i * step == r.gone ? w - 1.0 : w) : 0.0;
  }
}

// Sums over every `step`-th token from v on.
template <typename T>
__device__ __forceinline__ void sum_weights(const Rest<T>& r, int v, int end, int step, double& rest, double& whole) {
  rest = whole = 0.0;
  for (; v < end; v += 8 * step) {
    double a[8], b[8];
    if (r.q) weights_of<T, true, 8>(r, v, end, step, a, b);
    else weights_of<T, false, 8>(r, v, end, step, a, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      rest += a[i];
      whole += b[i];
    }
  }
}

// Sum over the lanes up to and with this one: shifts inside rows of 16 lanes, then the last lanes of rows to the rows behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ double shifted(double v) {        // 0 where nothing is shifted in
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, ROWS == 0xf);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, ROWS == 0xf);
  return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_scan_f64(double v) {
  v += shifted<0x111, 0xf>(v);
  v += shifted<0x112, 0xf>(v);
  v += shifted<0x114, 0xf>(v);
  v += shifted<0x118, 0xf>(v);
  v += shifted<0x142, 0xa>(v);
  v += shifted<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}

__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int taken, int hit) {
  const int j = threadIdx.x;
  if (j <= a.n) a.tokens[(long long)b * (a.n + 1) + j] = j < taken ? a.draft[b * a.d_bs + j] : j == taken ? hit : a.pad;
  if (j == 0) a.accepted[b] = taken;
}

__device__ __forceinline__ double border(const VerifyArgs& a, int b, double total) {
  return fmin(fmax((double)a.u[b * a.u_bs + a.n], 0.0), 1.0) * total;
}

// Sums before a thread's, over a workgroup of WAVES waves (s_w: scratch), and the sum of all.
template <int WAVES>
__device__ __forceinline__ double sum_before(double mine, int lane, int wave, double* s_w, double& total) {
  const double upto = wave_scan_f64(mine);
  if (lane == 63) s_w[wave] = upto;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += s_w[w];
    total += s_w[w];
  }
  return before + shifted<0x138, 0xf>(upto);                 // the lane before's
}

// The first token whose cumulative weight exceeds x, among [lo, hi) of this thread with the weights [before, before + mine);
// candidates of all threads meet in `hit` (the lowest stands).  Where rounding, or u = 1, leaves no token beyond x, the
// last with any weight stands in: it is entered behind all others.
template <typename T>
__device__ __forceinline__ void find_border(const Rest<T>& r, int lo, int hi, bool all, double before, double mine, double x, int* hit) {
  if (!(mine > 0.0) || before > x) return;
  int found = -1, last = -1;
  for (int v = lo; v < hi && found < 0; v += 8) {
    double a[8], b[8];
    if (r.q) weights_of<T, true, 8>(r, v, hi, 1, a, b);
    else weights_of<T, false, 8>(r, v, hi, 1, a, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double w = all ? b[i] : a[i];
      before += w;
      if (w > 0.0) {
        last = v + i;
        if (before > x && found < 0) found = v + i;
      }
    }
  }
  if (found >= 0) atomicMin(&hit[0], found);
  else if (last >= 0) atomicMax(&hit[1], last);
}
__device__ __forceinline__ void find_border(const double (&w)[8], int lo, double before, double mine, double x, int* hit) {
  if (!(mine > 0.0) || before > x) return;
  int found = -1, last = -1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    before += w[i];
    if (w[i] > 0.0) {
      last = lo + i;
      if (before > x && found < 0) found = lo + i;
    }
  }
  if (found >= 0) atomicMin(&hit[0], found);
  else atomicMax(&hit[1], last);
}
__device__ __forceinline__ int hit_of(const int* hit) { return hit[0] < 0x7fffffff ? hit[0] : max(hit[1], 0); }

// One workgroup per sequence, the whole row in registers: wave w holds U x 64 consecutive weights, U of them a lane.
template <typename T, int WAVES, int U>
__global__ __launch_bounds__(64 * WAVES) void verify_small_kernel(const VerifyArgs a) {
  __shared__ double s_rest[WAVES], s_whole[WAVES];
  __shared__ int s_hit[2];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int taken = taken_drafts<T>(a, b, lane);
  const Rest<T> r(a, b, taken);
  const int v0 = wave * U * 64 + lane;
  double w[U], full[U], rest = 0.0, whole = 0.0;
  if (r.q) weights_of<T, true, U>(r, v0, a.V, 64, w, full);
  else weights_of<T, false, U>(r, v0, a.V, 64, w, full);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    rest += w[i];
    whole += full[i];
  }
  rest = wave_scan_f64(rest);
  whole = wave_scan_f64(whole);
  if (lane == 63) {
    s_rest[wave] = rest;
    s_whole[wave] = whole;
  }
  if (threadIdx.x == 0) {
    s_hit[0] = 0x7fffffff;
    s_hit[1] = -1;                                           // a row without any weight: token 0
  }
  __syncthreads();
  double total = 0.0, before = 0.0, mine = 0.0;
#pragma unroll
  for (int x = 0; x < WAVES; ++x) total += s_rest[x];
  const bool all = !(total > 0.0);                           // nothing remains: the target's row as it is
  total = 0.0;
#pragma unroll
  for (int x = 0; x < WAVES; ++x) {
    const double sum = all ? s_whole[x] : s_rest[x];
    if (x < wave) before += sum;
    if (x == wave) mine = sum;
    total += sum;
  }
  const double x = border(a, b, total);
  if (total > 0.0 && total < INFINITY && mine > 0.0 && before <= x) {       // the same for every lane of a wave
    int found = -1, last = -1;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const double m = all ? full[i] : w[i], upto = before + wave_scan_f64(m);
      const unsigned long long hit = __ballot(m > 0.0 && upto > x), any = __ballot(m > 0.0);
      if (found < 0 && hit) found = i * 64 + __ffsll(hit) - 1;
      if (any) last = i * 64 + 63 - __clzll(any);
      before = lane_f64(upto, 63);
    }
    if (lane == 0) {
      if (found >= 0) atomicMin(&s_hit[0], wave * U * 64 + found);
      else if (last >= 0) atomicMax(&s_hit[1], wave * U * 64 + last);
    }
  }
  __syncthreads();
  write_tokens(a, b, taken, hit_of(s_hit));
}

// The border x in the piece [p0, p1) of a row, whose weights begin at `before`: an equal part for every thread of WAVES waves.
template <typename T, int WAVES>
__device__ __forceinline__ void find_in_piece(const Rest<T>& r, int p0, int p1, bool all, double before, double x, int lane,
                                              int wave, double* s_w, int* s_hit) {
  const int per = (p1 - p0 + 64 * WAVES - 1) / (64 * WAVES), lo = min(p0 + (int)threadIdx.x * per, p1), hi = min(lo + per, p1);
  double sum;
  if (per <= 8) {                                            // read once: 1 x 50265 8.0 us, read twice 8.5
    double w[8], full[8], mine = 0.0;
    if (r.q) weights_of<T, true, 8>(r, lo, hi, 1, w, full);
    else weights_of<T, false, 8>(r, lo, hi, 1, w, full);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = all ? full[i] : w[i];
      mine += w[i];
    }
    const double prior = sum_before<WAVES>(mine, lane, wave, s_w, sum);
    find_border(w, lo, before + prior, mine, x, s_hit);
  } else {
    double rest, whole;
    sum_weights(r, lo, hi, 1, rest, whole);
    const double mine = all ? whole : rest, prior = sum_before<WAVES>(mine, lane, wave, s_w, sum);
    find_border(r, lo, hi, all, before + prior, mine, x, s_hit);
  }
}

// One workgroup per sequence: a wave sums a contiguous piece of the row, then all of them look for the border in the piece
// that holds it.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void verify_draft_kernel(const VerifyArgs a) {
  __shared__ double s_rest[WAVES], s_whole[WAVES], s_w[WAVES];
  __shared__ int s_hit[2];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int taken = taken_drafts<T>(a, b, lane);
  const Rest<T> r(a, b, taken);
  const int piece = (a.V + WAVES - 1) / WAVES, w0 = min(wave * piece, a.V), w1 = min(w0 + piece, a.V);
  double rest, whole;
  sum_weights(r, w0 + lane, w1, 64, rest, whole);
  rest = wave_scan_f64(rest);
  whole = wave_scan_f64(whole);
  if (lane == 63) {
    s_rest[wave] = rest;
    s_whole[wave] = whole;
  }
  if (threadIdx.x == 0) {
    s_hit[0] = 0x7fffffff;
    s_hit[1] = -1;                                           // a row without any weight: token 0
  }
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += s_rest[w];
  const bool all = !(total > 0.0);                           // nothing remains: the target's row as it is
  if (all) {
    total = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += s_whole[w];
  }
  if (total > 0.0 && total < INFINITY) {                     // the same for every thread
    const double x = border(a, b, total);
    // the piece: the last one with weight that does not begin beyond x
    double run = 0.0, before = 0.0;
    int at = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const double mine = all ? s_whole[w] : s_rest[w];
      if (mine > 0.0 && run <= x) {
        at = w;
        before = run;
      }
      run += mine;
    }
    find_in_piece<T, WAVES>(r, min(at * piece, a.V), min(at * piece + piece, a.V), all, before, x, lane, wave, s_w, s_hit);
  }
  __syncthreads();
  write_tokens(a, b, taken, hit_of(s_hit));
}

// The same with a sequence's row over `pieces` workgroups: sums first ...
template <typename T>
__global__ __launch_bounds__(256) void verify_sum_kernel(const VerifyArgs a) {
  __shared__ double s_rest[4], s_whole[4];
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int taken = taken_drafts<T>(a, b, lane);
  const Rest<T> r(a, b, taken);
  const int piece = (a.V + a.pieces - 1) / a.pieces, lo = blockIdx.x * piece, hi = min(lo + piece, a.V);
  double rest, whole;
  sum_weights(r, lo + (int)threadIdx.x, hi, 256, rest, whole);
  rest = wave_scan_f64(rest);
  whole = wave_scan_f64(whole);
  if (lane == 63) {
    s_rest[wave] = rest;
    s_whole[wave] = whole;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double* to = a.sums + ((long long)b * a.pieces + blockIdx.x) * 2;
    to[0] = s_rest[0] + s_rest[1] + s_rest[2] + s_rest[3];
    to[1] = s_whole[0] + s_whole[1] + s_whole[2] + s_whole[3];
    if (blockIdx.x == 0) a.accepted[b] = taken;
  }
}

// ... then, per sequence, the piece that holds the border (at most 64 of them: a lane each) and the border in it.
template <typename T>
__global__ __launch_bounds__(256) void verify_find_kernel(const VerifyArgs a) {
  __shared__ double s_w[4];
  __shared__ int s_hit[2];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int taken = a.accepted[b];                           // from the sums' kernel
  const Rest<T> r(a, b, taken);
  double rest = 0.0, whole = 0.0;
  if (lane < a.pieces) {
    const double* from = a.sums + ((long long)b * a.pieces + lane) * 2;
    rest = from[0];
    whole = from[1];
  }
  double upto = wave_scan_f64(rest), total = lane_f64(upto, 63);
  const bool all = !(total > 0.0);                           // nothing remains: the target's row as it is
  if (all) {
    rest = whole;
    upto = wave_scan_f64(rest);
    total = lane_f64(upto, 63);
  }
  const double x = border(a, b, total);
  // sums of lanes are associated differently, so an upto may lie a rounding beyond the total, or under the one before it
  const unsigned long long past = __ballot(rest > 0.0 && upto > x), any = __ballot(rest > 0.0);
  if (threadIdx.x == 0) {
    s_hit[0] = 0x7fffffff;
    s_hit[1] = -1;                                           // a row without any weight: token 0
  }
  if (any && total > 0.0 && total < INFINITY) {              // the same for every thread of the workgroup
    const int at = past ? __ffsll(past) - 1 : 63 - __clzll(any);
    const double before = at ? fmin(lane_f64(upto, at - 1), x) : 0.0;
    const int piece = (a.V + a.pieces - 1) / a.pieces, p0 = at * piece, p1 = min(p0 + piece, a.V);
    find_in_piece<T, 4>(r, p0, p1, all, before, x, lane, wave, s_w, s_hit);
  }
  __syncthreads();
  write_tokens(a, b, taken, hit_of(s_hit));
}

template <typename T>
static void launch_verify(const VerifyArgs& a, hipStream_t stream) {
  if (a.pieces > 1) {
    hipLaunchKernelGGL(verify_sum_kernel<T>, dim3(a.pieces, a.B), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(verify_find_kernel<T>, dim3(a.B), dim3(256), 0, stream, a);
  } else if (a.V > 8192) {
    hipLaunchKernelGGL((verify_draft_kernel<T, 16>), dim3(a.B), dim3(1024), 0, stream, a);
  } else if (a.V > 1024) {
    hipLaunchKernelGGL((verify_small_kernel<T, 16, 8>), dim3(a.B), dim3(1024), 0, stream, a);
  } else {
    hipLaunchKernelGGL((verify_small_kernel<T, 4, 4>), dim3(a.B), dim3(256), 0, stream, a);
  }
}

// draft: [B, n] int32, p: [B, n + 1, V], q: [B, n, V] or null, u: [B, n + 1] fp32, counts: [B] or null;
// tokens: [B, n + 1], accepted: [B].  dtype: 0 bf16, 1 fp16, 2 fp32.  pieces: workgroups a row is spread over (1 .. 64);
// sums: [B][pieces][2] doubles where pieces > 1.
extern "C" int dlamd_verify_draft(const void* draft, long long d_bs, const void* p, long long p_bs, long long p_ns,
                                  const void* q, long long q_bs, long long q_ns, const void* u, long long u_bs,
                                  const void* counts, void* tokens, void* accepted, void* sums, long long sums_doubles, int pieces, int B, int n,
                                  int V, int pad, int dtype, hipStream_t stream) {
  if (B <= 0) return 0;
  if (n < 0 || n > 63 || V <= 0 || V >= 0x40000000 || B >= 1 << 22) return -1;      // a launch has fewer than 2^32 threads
  if (pieces < 1 || pieces > 64 || (pieces > 1 && (B > 65535 || !sums || ((uintptr_t)sums & 7) || sums_doubles < 2LL * B * pieces))) return -3;
  VerifyArgs a{(const int*)draft, p, q, (const float*)u, (const int*)counts, (int*)tokens, (int*)accepted, d_bs, p_bs, p_ns,
               q_bs, q_ns, u_bs, (double*)sums, B, n, V, pad, pieces};
  if (dtype == 0) launch_verify<bf16_t>(a, stream);
  else if (dtype == 1) launch_verify<f16_t>(a, stream);
  else if (dtype == 2) launch_verify<float>(a, stream);
  else return -2;
  return DLAMD_CHECK_LAUNCH();
}
