// Attention of one or a few new tokens per sequence over a paged key / value cache.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the visible positions j of the sequence, one pass over keys and values with
// the running maximum m and sum l of the softmax (a new maximum rescales what is summed so far by exp(m_old - m_new)).
// A position is visible when it is below the row's limit and its page exists; keys and values of other positions
// are never used in arithmetic, whatever they hold.  A row without visible positions is 0, its log-sum-exp -inf.
//
// The cost is reading the cache once, so everything serves loads in flight:
//   * The n new tokens x (heads / kv_heads) query heads that read one key head are the rows of ONE problem (16, 32 or 64
//     per workgroup): a key is fetched once for all of them and the products run on matrix instructions, padded to 16.
//   * A wave takes tiles of 32 keys by itself, straight from memory into the operand registers, the next tile's loads in
//     flight while it computes; no LDS, no barrier until the four waves of a workgroup join their (m, l, o).
//   * S^T = K Q^T: A = K (a lane holds 8 dimensions of one key, as they lie in memory), so a lane's accumulators are 4 keys
//     of ONE query.  O^T = V^T P^T: B = P^T straight from those accumulators, with the keys in the order they hold:
//     operand slot 8 g + 4 t + j of lane group g is key 16 t + 4 g + j.  A = V^T: a lane loads the same D / 16 consecutive
//     dimensions of its 8 keys (16 lanes cover a key's row: whole lines) and turns the block in registers; output tile i
//     then holds dimension (D / 16) r + i in row r, which leaves a lane with D / 4 consecutive dimensions of one query.
//   * P goes into the products as two 16-bit halves, hi + lo: one rounding to 16 bits would cost as much accuracy as the
//     result's own rounding, and the second product hides behind the loads.
//   * Long sequences are split into chunks; each writes its (m, l, o) in 32 bits and a second kernel joins them.  The chunk
//     is fixed by the host from the longest length a sequence may have, so a short sequence has few chunks and the
//     workgroups of the others end at once.
#include "common.h"

typedef _Float16 f16_t;

struct PagedAttArgs {
  const void *q, *kp, *vp;
  void* o;
  float* lse;
  float* part;                                               // [units][splits][rows][D + 2]: o, then m, l
  const int *table, *lens;
  long long q_bs, q_ns, q_hs;
  long long k_ps, v_ps, t_bs;                                // page strides of the cache in bytes; table rows in entries
  int k_ss, k_hs, v_ss, v_hs;                                // slot / head strides in bytes
  int B, n, Hq, Hkv, page, width, pages, causal;
  int splits, chunk, groups;                                 // chunk: keys per split; groups: row groups per (b, kv head)
  uint32_t page_magic;                                       // ceil(2^32 / (page / 16))
  float scale2;                                              // scale * log2(e)
};

#define ROW_NONE (-3.4028234e38f)                            // running maximum of nothing: finite, so differences stay numbers
#define LN2 0.6931471805599453f

template <typename T> struct Mat;
template <> struct Mat<bf16_t> {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<f16_t> {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// Where the two halves (16 keys, one page each) of a tile of 32 keys lie.
struct Place {
  const char *k[2], *v[2];                                   // the half's first key / value row
  int last[2];                                               // last readable row of the half
  bool ok[2];                                                // the half's page exists and some row sees it
};

// Page of the 16 keys at `key` (beyond the limit: none).  Uniform over the wave: the entry comes by a scalar load.
__device__ __forceinline__ int page_of(const PagedAttArgs& p, const int* row, int key, int limit) {
  const int unit = key >> 4;
  const int pi = p.page_magic ? (int)__umulhi((uint32_t)unit, p.page_magic) : unit;
  return key < limit ? row[pi] : -1;
}

// Rows that no one sees are not skipped but replaced by rows that are there (the limit's last one, or page 0): loads then
// have no branches, and what they bring is masked (keys) or cleared (values) afterwards.  kh, vh: the head's first byte.
__device__ __forceinline__ void find_tile(Place& t, const PagedAttArgs& p, const char* kh, const char* vh, int pid0, int pid1,
                                          int k0, int limit) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int key = k0 + 16 * h, pid = h ? pid1 : pid0;
    const int unit = key >> 4;
    const int pi = p.page_magic ? (int)__umulhi((uint32_t)unit, p.page_magic) : unit;
    t.ok[h] = pid >= 0 && pid < p.pages;
    const int at = t.ok[h] ? pid : 0, slot = t.ok[h] ? key - pi * p.page : 0;
    t.k[h] = kh + at * p.k_ps + slot * p.k_ss;
    t.v[h] = vh + at * p.v_ps + slot * p.v_ss;
    t.last[h] = t.ok[h] ? min(15, limit - 1 - key) : 15;
  }
}

template <int D>
__device__ __forceinline__ void load_k(u32x4 (&k)[2][D / 32], const PagedAttArgs& p, const Place& t, int r, int g) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t off = __umul24(min(r, t.last[h]), p.k_ss) + 16 * g;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) k[h][s] = *reinterpret_cast<const u32x4*>(t.k[h] + off + 64 * s);
  }
}

template <int D>
__device__ __forceinline__ void load_v(uint32_t (&v)[8][D / 32], const PagedAttArgs& p, const Place& t, int r, int g) {
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const uint32_t off = __umul24(min(4 * g + (s & 3), t.last[s >> 2]), p.v_ss) + D / 8 * r;
    const char* b = t.v[s >> 2];
    if (D == 128) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(b + off);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[s][i] = x[i];
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(b + off);
      v[s][0] = x[0];
      v[s][1] = x[1];
    }
  }
}

template <typename T, int D, int MT>
struct Rows {                                                // what a wave holds of its rows
  f32x4 o[MT][D / 16];
  float m[MT], l[MT];
  int lim[MT];
  typename Mat<T>::x8 q[MT][D / 32];
};

// Scores of one tile (in units of log 2), -inf where a row does not see the key.
template <typename T, int D, int MT>
__device__ __forceinline__ void scores(f32x4 (&x)[MT][2], const Rows<T, D, MT>& w, const u32x4 (&k)[2][D / 32], const Place& t,
                                       const PagedAttArgs& p, int k0, int g) {
  typedef typename Mat<T>::x8 x8;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int seen = (t.ok[h] ? w.lim[mt] : 0) - (k0 + 16 * h + 4 * g);
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) s = Mat<T>::mul(__builtin_bit_cast(x8, k[h][c]), w.q[mt][c], s);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[mt][h][j] = j < seen ? s[j] * p.scale2 : -INFINITY;
    }
}

// Scores to weights, against the running maximum.
template <typename T, int D, int MT>
__device__ __forceinline__ void weights(typename Mat<T>::x8 (&hi)[MT], typename Mat<T>::x8 (&lo)[MT], Rows<T, D, MT>& w,
                                        const f32x4 (&x)[MT][2]) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float top = ROW_NONE;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(x[mt][0][j], x[mt][1][j]));
    if (__any(top > w.m[mt])) {                              // rare once the largest scores have been seen
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float m = fmaxf(w.m[mt], top);
      const float a = __builtin_amdgcn_exp2f(w.m[mt] - m);
      w.m[mt] = m;
      w.l[mt] *= a;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) w.o[mt][i][j] *= a;
    }
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = __builtin_amdgcn_exp2f(x[mt][h][j] - w.m[mt]);
        sum += e;
        const T eh = (T)e;
        hi[mt][4 * h + j] = eh;
        lo[mt][4 * h + j] = (T)(e - (float)eh);
      }
    w.l[mt] += sum;                                          // this lane's keys; the four lane groups join at the end
  }
}

// Weights times values into the rows' sums.
template <typename T, int D, int MT>
__device__ __forceinline__ void add_values(Rows<T, D, MT>& w, uint32_t (&v)[8][D / 32], const typename Mat<T>::x8 (&hi)[MT],
                                           const typename Mat<T>::x8 (&lo)[MT], const Place& t, bool all, int k0,
                                           int limit_all, int limit, int g, bool& odd) {
  typedef typename Mat<T>::x8 x8;
  if (!all) {
    // Rows of later tokens see keys that rows of earlier ones do not.  A product of a hidden key's weight, 0, and a value
    // that is no finite number would be NaN, so such values leave the product here and are added row by row at the end.
    constexpr uint32_t EXP = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int key = k0 + 16 * (s >> 2) + 4 * g + (s & 3);
      const bool none = !t.ok[s >> 2] || key >= limit, some = key >= limit_all;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        if (none) v[s][c] = 0u;
        uint32_t bad = 0u;
        if (some && (v[s][c] & EXP) == EXP) bad = 0xffffu;
        if (some && ((v[s][c] >> 16) & EXP) == EXP) bad |= 0xffff0000u;
        v[s][c] &= ~bad;
        odd |= bad != 0u;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    u32x4 a;                                                 // dimension (D / 16) r + i of the lane's 8 keys
#pragma unroll
    for (int c = 0; c < 4; ++c)
      a[c] = __builtin_amdgcn_perm(v[2 * c + 1][i >> 1], v[2 * c][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      w.o[mt][i] = Mat<T>::mul(__builtin_bit_cast(x8, a), hi[mt], w.o[mt][i]);
      w.o[mt][i] = Mat<T>::mul(__builtin_bit_cast(x8, a), lo[mt], w.o[mt][i]);
    }
  }
}

// What add_values left out: values that are no finite numbers, at the (less than n) positions that some rows see and others
// do not.  Never in sane use: the weight is computed again, element by element.
template <typename T, int D, int MT>
__device__ __forceinline__ void add_odd_values(Rows<T, D, MT>& w, const PagedAttArgs& p, const int* row, int b, int hk, int row0,
                                               int R, int G, int kb, int wave, int limit_all, int limit, int r, int g) {
  constexpr uint32_t EXP = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
#pragma unroll 1
  for (int key = max(kb, limit_all); key < limit; ++key) {
    if ((((key - kb) >> 5) & 3) != wave) continue;
    const int pi = key / p.page, pid = row[pi];
    if (pid < 0 || pid >= p.pages) continue;
    const long long slot = key - pi * p.page;
    const T* kr = (const T*)((const char*)p.kp + pid * p.k_ps + slot * p.k_ss + (long long)hk * p.k_hs);
    const T* vr = (const T*)((const char*)p.vp + pid * p.v_ps + slot * p.v_ss + (long long)hk * p.v_hs) + D / 4 * g;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int at = row0 + 16 * mt + r, i = at / G, h = hk * G + at - i * G;
      if (at >= R || key >= w.lim[mt]) continue;
      const T* qr = (const T*)p.q + b * p.q_bs + i * p.q_ns + h * p.q_hs;
      float x = 0.f;
#pragma unroll 1
      for (int d = 0; d < D; ++d) x += (float)qr[d] * (float)kr[d];
      const float e = __builtin_amdgcn_exp2f(x * p.scale2 - w.m[mt]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {                   // the lane's sums: dimensions D / 4 g .. of its query
          const uint32_t bits = *reinterpret_cast<const uint16_t*>(vr + D / 16 * j + c);
          if ((bits & EXP) == EXP) w.o[mt][c][j] += e * (float)vr[D / 16 * j + c];
        }
    }
  }
}

template <typename T, int D, int MT>
__global__ __launch_bounds__(256, MT == 1 ? 3 : MT == 2 ? 2 : 1) void paged_attention_kernel(const PagedAttArgs p) {
  typedef typename Mat<T>::x8 x8;
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ float s_o[4][16][D + 4];                        // + 4: lanes of one group write 16 rows at once
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  int u = blockIdx.x;
  const int split = u % p.splits;
  u /= p.splits;
  const int group = u % p.groups, bh = u / p.groups;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int G = p.Hq / p.Hkv, R = p.n * G, row0 = group * 16 * MT;
  const int kept = p.lens[b];
  const int cap = p.width * p.page;
  const int base = kept < 0 ? 0 : min(kept, cap), more = kept >= 0 && p.causal;
  // limits of the group's first and last row; a chunk ends the last split only with the sequence
  const int rl = min(row0 + 16 * MT, R) - 1;
  const int limit_all = min(base + (more ? row0 / G + 1 : 0), cap);
  int limit = p.pages > 0 ? min(base + (more ? rl / G + 1 : 0), cap) : 0;
  const int kb = split * p.chunk;
  if (split > 0 && kb >= limit) return;                      // the join knows which chunks exist
  if (split < p.splits - 1) limit = min(limit, kb + p.chunk);

  Rows<T, D, MT> w;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + r;
    const int i = row / G, h = hk * G + row - i * G;
    w.lim[mt] = row < R ? min(min(base + (more ? i + 1 : 0), cap), limit) : 0;
    w.m[mt] = ROW_NONE;
    w.l[mt] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      u32x4 t = {0u, 0u, 0u, 0u};
      if (row < R) t = *reinterpret_cast<const u32x4*>((const T*)p.q + b * p.q_bs + i * p.q_ns + h * p.q_hs + 32 * c + 8 * g);
      w.q[mt][c] = __builtin_bit_cast(x8, t);
    }
#pragma unroll
    for (int i2 = 0; i2 < D / 16; ++i2) w.o[mt][i2] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The next tile's keys are fetched into the registers of this one's as soon as the scores have been taken, its values
  // after the products: at any time a wave has most of a tile in flight, and three waves fit a SIMD.
  const int* row = p.table + b * p.t_bs;
  const char *kh = (const char*)p.kp + (long long)hk * p.k_hs, *vh = (const char*)p.vp + (long long)hk * p.v_hs;
  int k0 = kb + 32 * wave;
  bool odd = false;
  if (k0 < limit) {
    u32x4 k[2][D / 32];
    uint32_t v[8][D / 32];
    Place at;
    find_tile(at, p, kh, vh, page_of(p, row, k0, limit), page_of(p, row, k0 + 16, limit), k0, limit);
    load_k<D>(k, p, at, r, g);
    load_v<D>(v, p, at, r, g);
    int pid0 = page_of(p, row, k0 + 128, limit), pid1 = page_of(p, row, k0 + 144, limit);
    while (true) {
      const bool all = k0 + 32 <= limit_all && k0 + 32 <= limit && at.ok[0] && at.ok[1];
      const int k1 = k0 + 128;
      f32x4 x[MT][2];
      scores<T, D, MT>(x, w, k, at, p, k0, g);
      Place next;
      if (k1 < limit) {
        find_tile(next, p, kh, vh, pid0, pid1, k1, limit);
        load_k<D>(k, p, next, r, g);
        pid0 = page_of(p, row, k1 + 128, limit);
        pid1 = page_of(p, row, k1 + 144, limit);
      }
      x8 hi[MT], lo[MT];
      weights<T, D, MT>(hi, lo, w, x);
      add_values<T, D, MT>(w, v, hi, lo, at, all, k0, limit_all, limit, g, odd);
      if (k1 >= limit) break;
      load_v<D>(v, p, next, r, g);
      at = next;
      k0 = k1;
    }
  }
  if (__any(odd)) add_odd_values<T, D, MT>(w, p, row, b, hk, row0, R, G, kb, wave, limit_all, limit, r, g);
  // join the four waves, 16 rows at a time
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float l = w.l[mt];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (mt) __syncthreads();
    if (g == 0) {
      s_m[wave][r] = w.m[mt];
      s_l[wave][r] = l;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < D / 16; i += 4) {
        const f32x4 t = {w.o[mt][i][j], w.o[mt][i + 1][j], w.o[mt][i + 2][j], w.o[mt][i + 3][j]};
        *reinterpret_cast<f32x4*>(&s_o[wave][r][(D / 16) * (4 * g + j) + i]) = t;
      }
    __syncthreads();
    // thread: row threadIdx / 16, D / 16 dimensions
    const int row_ = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16), row = row0 + 16 * mt + row_;
    if (row < R) {
      const float m = fmaxf(fmaxf(s_m[0][row_], s_m[1][row_]), fmaxf(s_m[2][row_], s_m[3][row_]));
      float f[4], sum = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        f[x] = __builtin_amdgcn_exp2f(s_m[x][row_] - m);
        sum += f[x] * s_l[x][row_];
      }
      float o[D / 16];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        o[d] = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[d] += f[x] * s_o[x][row_][d0 + d];
      }
      const int i = row / G, h = hk * G + row - i * G;
      const long long at = ((long long)b * p.n + i) * p.Hq + h;
      if (p.splits == 1) {
        const float inv = 1.f / sum;
        T t[D / 16];
#pragma unroll
        for (int d = 0; d < D / 16; ++d) t[d] = (T)(sum == 0.f ? 0.f : o[d] * inv);   // sum is NaN where a score is
        T* dst = (T*)p.o + at * D + d0;
#pragma unroll
        for (int d = 0; d < D / 16; d += 4) *reinterpret_cast<u32x2*>(dst + d) = *reinterpret_cast<u32x2*>(t + d);
        if (p.lse && d0 == 0) p.lse[at] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * LN2;
      } else {
        float* dst = p.part + ((long long)at * p.splits + split) * (D + 4);
#pragma unroll
        for (int d = 0; d < D / 16; d += 4) *reinterpret_cast<f32x4*>(dst + d0 + d) = f32x4{o[d], o[d + 1], o[d + 2], o[d + 3]};
        if (d0 == 0) {
          dst[D] = m;
          dst[D + 1] = sum;
        }
      }
    }
  }
}

// One workgroup per row: joins the chunks of its sequence.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(const PagedAttArgs p, int rows_per_group) {
  constexpr int TD = D / 4, SL = 256 / TD;                   // threads per chunk (4 dimensions each), chunks side by side
  __shared__ float s_o[SL][D];
  __shared__ float s_l[SL], s_m[SL];
  const long long at = blockIdx.x;
  const int h = (int)(at % p.Hq), i = (int)((at / p.Hq) % p.n), b = (int)(at / ((long long)p.Hq * p.n));
  const int G = p.Hq / p.Hkv;
  const int kept = p.lens[b], cap = p.width * p.page;
  const int base = kept < 0 ? 0 : min(kept, cap), more = kept >= 0 && p.causal;
  // as many chunks as the row's group has: the limit of the group's last row
  const int row = i * G + h % G, rl = min((row / rows_per_group + 1) * rows_per_group, p.n * G) - 1;
  const int limit = p.pages > 0 ? min(base + (more ? rl / G + 1 : 0), cap) : 0;
  const int have = max(1, min(p.splits, (limit + p.chunk - 1) / p.chunk));
  const int d = (threadIdx.x % TD) * 4, sl = threadIdx.x / TD;
  const float* src = p.part + at * p.splits * (D + 4);
  float m = ROW_NONE, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = sl; s < have; s += SL) {
    const float* q = src + (long long)s * (D + 4);
    const float ms = q[D], ls = q[D + 1], mn = fmaxf(m, ms);
    const f32x4 os = *reinterpret_cast<const f32x4*>(q + d);
    const float a = __builtin_amdgcn_exp2f(m - mn), c = __builtin_amdgcn_exp2f(ms - mn);
    l = l * a + ls * c;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * a + os[j] * c;
    m = mn;
  }
  *reinterpret_cast<f32x4*>(&s_o[sl][d]) = o;
  if (d == 0) {
    s_l[sl] = l;
    s_m[sl] = m;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float top = ROW_NONE, sum = 0.f, v = 0.f;
#pragma unroll
    for (int x = 0; x < SL; ++x) top = fmaxf(top, s_m[x]);
#pragma unroll
    for (int x = 0; x < SL; ++x) {
      const float f = __builtin_amdgcn_exp2f(s_m[x] - top);
      sum += f * s_l[x];
      v += f * s_o[x][threadIdx.x];
    }
    ((T*)p.o)[at * D + threadIdx.x] = (T)(sum == 0.f ? 0.f : v / sum);
    if (p.lse && threadIdx.x == 0) p.lse[at] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * LN2;
  }
}

template <typename T, int D, int MT>
static void launch(const PagedAttArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((paged_attention_kernel<T, D, MT>), dim3((unsigned)(a.B * a.Hkv * a.groups * a.splits)), dim3(256), 0, stream, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((paged_attention_join_kernel<T, D>), dim3((unsigned)(a.B * a.n * a.Hq)), dim3(256), 0, stream, a, 16 * MT);
}
template <typename T, int D>
static void launch_rows(const PagedAttArgs& a, int mt, hipStream_t stream) {
  if (mt == 1) launch<T, D, 1>(a, stream);
  else if (mt == 2) launch<T, D, 2>(a, stream);
  else launch<T, D, 4>(a, stream);
}

// q: [B, n, Hq, D] (strides given), o: [B, n, Hq, D] contiguous, lse: [B, n, Hq] or null.  dtype: 0 bf16, 1 fp16.
// splits chunks of `chunk` keys (the last one takes the rest); part: [B n Hq][splits][D + 4] floats where splits > 1.
extern "C" int dlamd_paged_attention(const void* q, long long q_bs, long long q_ns, long long q_hs, const void* kp,
                                     long long kp_ps, long long kp_ss, long long kp_hs, const void* vp, long long vp_ps,
                                     long long vp_ss, long long vp_hs, const void* table, long long t_bs,
                                     const void* lens, void* o, void* lse, void* part, int splits, int chunk, int B, int n,
                                     int Hq, int Hkv, int D, int page, int width, int pages, int causal, float scale,
                                     int dtype, hipStream_t stream) {
  if (B <= 0 || n <= 0 || Hq <= 0) return 0;
  if (Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128)) return -1;
  if (page <= 0 || page % 16 != 0 || width < 0 || pages < 0) return -2;
  if ((q_bs | q_ns | q_hs | kp_ps | kp_ss | kp_hs | vp_ps | vp_ss | vp_hs) % 8 != 0) return -3;
  if (((uintptr_t)q | (uintptr_t)kp | (uintptr_t)vp | (uintptr_t)o) & 15) return -4;
  // a lane's offset inside 16 slots is a 24-bit product, a head's and a page's inside one page 32 bits
  const long long sl[4] = {kp_ss * 2, vp_ss * 2, kp_hs * 2, vp_hs * 2};
  if (sl[0] < 0 || sl[1] < 0 || sl[0] >= (1 << 24) || sl[1] >= (1 << 24) || sl[2] < 0 || sl[3] < 0 || sl[2] > 0x7fffffff ||
      sl[3] > 0x7fffffff || page * sl[0] > 0x7fffffff || page * sl[1] > 0x7fffffff)
    return -11;
  // positions are 32-bit; the page of a position is a multiplication, exact while units * (page / 16) < 2^32
  if ((long long)width * page > 0x7fffff00LL || (long long)width * (page / 16) * (page / 16) >= (1LL << 32)) return -5;
  if (dtype != 0 && dtype != 1) return -6;
  if (splits < 1 || chunk < 128 || chunk % 128 != 0 || (long long)(splits - 1) * chunk > 0x7fffff00LL) return -7;
  if (splits > 1 && (!part || ((uintptr_t)part & 15))) return -8;
  const int R = n * (Hq / Hkv);
  if ((long long)n * Hq > 0x7fffffffLL || (long long)B * n * Hq > 0x7fffffffLL) return -9;
  const int mt = R <= 16 ? 1 : R <= 32 ? 2 : 4;
  const int groups = (R + 16 * mt - 1) / (16 * mt);
  if ((long long)B * Hkv * groups * splits > 0x7fffffffLL) return -10;
  const uint32_t units = (uint32_t)(page / 16);
  const uint32_t magic = units == 1 ? 0u : (uint32_t)((0x100000000ULL + units - 1) / units);
  PagedAttArgs a{q, kp, vp, o, (float*)lse, (float*)part, (const int*)table, (const int*)lens, q_bs, q_ns, q_hs,
                 kp_ps * 2, vp_ps * 2, t_bs, (int)sl[0], (int)sl[2], (int)sl[1], (int)sl[3], B, n, Hq, Hkv, page, width, pages, causal,
                 splits, chunk, groups, magic, scale * 1.4426950408889634f};
  if (dtype == 0 && D == 64) launch_rows<bf16_t, 64>(a, mt, stream);
  if (dtype == 0 && D == 128) launch_rows<bf16_t, 128>(a, mt, stream);
  if (dtype == 1 && D == 64) launch_rows<f16_t, 64>(a, mt, stream);
  if (dtype == 1 && D == 128) launch_rows<f16_t, 128>(a, mt, stream);
  return DLAMD_CHECK_LAUNCH();
}
