// Attention of one or a few new tokens per sequence over a paged key / value cache.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the visible positions j of the sequence, one pass over keys and values with
// the running maximum m and sum l of the softmax (a new maximum rescales what is summed so far by exp(m_old - m_new)).
// A position is visible when it is below the row's limit and its page exists; keys and values of other positions
// are never used in arithmetic, whatever they hold.  A row without visible positions is 0, its log-sum-exp -inf.
//
// The cost is reading the cache once, so everything serves loads in flight:
//   * The n new tokens x (heads / kv_heads) query heads that read one key head are the rows of ONE problem (up to 48 per
//     workgroup, further groups on the same die): a key is fetched once for all of them and the products run on matrix
//     instructions, padded to 16.
//   * A wave takes tiles of 32 keys by itself, straight from memory into the operand registers, the next tile's loads in
//     flight while it computes; no LDS, no barrier until the four waves of a workgroup join their (m, l, o).
//   * S^T = K Q^T: A = K (a lane holds 8 dimensions of one key, as they lie in memory), so a lane's accumulators are 4 keys
//     of ONE query.  O^T = V^T P^T: B = P^T straight from those accumulators, with the keys in the order they hold:
//     operand slot 8 g + 4 t + j of lane group g is key 16 t + 4 g + j.  A = V^T: a lane loads the same D / 16 consecutive
//     dimensions of its 8 keys (16 lanes cover a key's row: whole lines) and turns the block in registers; output tile i
//     then holds dimension (D / 16) r + i in row r, which leaves a lane with D / 4 consecutive dimensions of one query.
//   * P goes into the products as two 16-bit halves, hi + lo: one rounding to 16 bits would cost as much accuracy as the
//     result's own rounding, and the second product hides behind the loads.  bf16 halves keep 16 bits of every weight.  fp16
//     ends at 2^-24, so weights (and l, and o) are 2^14 times as large there: 22 bits down to 2^-18 of the largest weight,
//     and nothing above 2^-38 of it is lost (unshifted, truncation took 3 % of weights of e^-14 of the largest).
//   * Long caches are cut into parts of as many tiles (of 128 keys) as give every compute unit its share.  The size of a
//     part is computed on the device from the lengths of the whole batch, so neither one long sequence nor a batch of very
//     different lengths leaves compute units idle, and a captured call adapts while lengths grow.  A part is written as
//     (m, l, o) in 32 bits and a second kernel joins the parts.  Short caches (and many of them) take one workgroup each.
//
// 100003 positions, 32 / 8 heads of 128: 83 us, 5.0 TB/s, what a copy reaches.  64 x 577 positions, 16 heads of 64: 34.0 us,
// 4.5 TB/s.  12 x 5 tokens over ragged caches of up to 8009: 25.5 us, 2.3 TB/s; a wave has three or four tiles there, and what
// precedes its first and follows its last one (page table, join of the waves, 5 us for the parts) is as long as their stream
// and hidden by nothing: with three row tiles of 128 dimensions a wave has 361 registers and its SIMD to itself.
#include "common.h"
#include "decode_abi.h"

typedef _Float16 f16_t;

// Page table and lengths: constant memory to the compiler (the kernel's stores do not change them), so entries at uniform
// places come by scalar loads, which do not wait for the tiles in flight.
typedef const int __attribute__((address_space(4)))* const_i32;

struct PagedAttArgs {
  const void *q, *kp, *vp;
  void* o;
  float* lse;
  float* part;                                               // [workgroups][rows][D + 4]: o, then m, l; the first row's next
                                                             // word: tiles of a part
  const int *table, *lens;
  long long q_bs, q_ns, q_hs;
  long long k_ps, k_hs, v_ps, v_hs, t_bs;                    // page / head strides of the cache in bytes; table rows in entries
  int k_ss, v_ss;                                            // slot strides in bytes
  int B, n, Hq, Hkv, page, width, pages, causal;
  int groups, rows, share, least;                            // row groups per (b, kv head), rows per group; workgroups to deal
                                                             // tiles out to (0: one for each problem), least tiles of a part
  uint32_t page_magic;                                       // ceil(2^32 / (page / 16))
  float scale2;                                              // |scale| log2(e), above 0: -inf stays -inf
  uint32_t flip;                                             // sign bits to turn in q where the scale is negative
};

#define ROW_NONE (-3.4028234e38f)                            // running maximum (of unscaled scores) of nothing: finite, so differences
                                                             // stay numbers
#define LN2 0.6931471805599453f

// mul: a 16x16x32 product; split: two weights as 16-bit halves hi + lo (hi may be rounded either way, lo makes up for it); UP:
// weights are 2^UP exp(score - maximum), DOWN is 2^-UP.
template <typename T> struct Mat;
template <> struct Mat<bf16_t> {
  static constexpr float UP = 0.f, DOWN = 1.f;
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const x2 h = {(__bf16)a, (__bf16)b};
    hi = __builtin_bit_cast(uint32_t, h);
    const x2 l = {(__bf16)(a - __builtin_bit_cast(float, hi << 16)), (__bf16)(b - __builtin_bit_cast(float, hi & 0xffff0000u))};
    lo = __builtin_bit_cast(uint32_t, l);
  }
  static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<f16_t> {
  static constexpr float UP = 14.f, DOWN = 1.f / 16384.f;
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a - (float)h[0], b - (float)h[1]));
  }
  static __device__ __forceinline__ f32x4 mul(x8 a, x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

typedef const char __attribute__((address_space(1)))* global_p;         // global memory, said so: no generic loads
typedef const u32x4 __attribute__((address_space(1)))* global_u32x4;
typedef const u32x2 __attribute__((address_space(1)))* global_u32x2;

// What stands in for the rows of a page that does not exist: a row of zeros, read 16 times.
__device__ const u32x4 k_zero_row[16] = {};

// Where the two halves (16 keys, one page each) of a tile of 32 keys lie.
struct Place {
  global_p k[2], v[2];                                       // the half's first key / value row
  int ks[2], vs[2];                                          // bytes from row to row, 0 for the row of zeros
  int last[2];                                               // last row of the half below the limit
  bool ok[2];                                                // the half's page exists and some row sees it
};

// Page of the 16 keys at `key`, whether or not they lie below the limit (behind the table: its last entry).  Uniform over the
// wave: the entry comes by a scalar load, without a branch.
__device__ __forceinline__ int page_of(const PagedAttArgs& p, const_i32 row, int key) {
  const int unit = key >> 4;
  const int pi = p.page_magic ? (int)__umulhi((uint32_t)unit, p.page_magic) : unit;
  return row[min(pi, p.width - 1)];
}

// Rows that no one sees are not skipped but replaced by rows that are there (the limit's last one, or zeros for a missing
// page): loads then have no branches.  kh, vh: the head's first byte.
__device__ __forceinline__ void find_tile(Place& t, const PagedAttArgs& p, global_p kh, global_p vh, int pid0, int pid1, int k0,
                                          int limit) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int key = k0 + 16 * h, pid = h ? pid1 : pid0;
    const int unit = key >> 4;
    const int pi = p.page_magic ? (int)__umulhi((uint32_t)unit, p.page_magic) : unit;
    const int slot = key - pi * p.page;
    t.ok[h] = key < limit && pid >= 0 && pid < p.pages;
    t.k[h] = t.ok[h] ? kh + pid * p.k_ps + slot * p.k_ss : (global_p)k_zero_row;
    t.v[h] = t.ok[h] ? vh + pid * p.v_ps + slot * p.v_ss : (global_p)k_zero_row;
    t.ks[h] = t.ok[h] ? p.k_ss : 0;
    t.vs[h] = t.ok[h] ? p.v_ss : 0;
    t.last[h] = limit - 1 - key;
  }
}

// TAIL: the tile may reach beyond the limit.
template <int D, bool TAIL>
__device__ __forceinline__ void load_k(u32x4 (&k)[2][D / 32], const Place& t, int r, int g) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t off = __umul24(TAIL && t.ok[h] ? min(r, t.last[h]) : r, t.ks[h]) + 16 * g;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) k[h][s] = *(global_u32x4)(t.k[h] + off + 64 * s);
  }
}

template <int D, bool TAIL>
__device__ __forceinline__ void load_v(uint32_t (&v)[8][D / 32], const Place& t, int r, int g) {
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int row = 4 * g + (s & 3), h = s >> 2;
    const uint32_t off = __umul24(TAIL && t.ok[h] ? min(row, t.last[h]) : row, t.vs[h]) + D / 8 * r;
    if (D == 128) {
      const u32x4 x = *(global_u32x4)(t.v[h] + off);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[s][i] = x[i];
    } else {
      const u32x2 x = *(global_u32x2)(t.v[h] + off);
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

// Scores of one tile before scaling, -inf where a row does not see the key.
template <typename T, int D, int MT, bool TAIL>
__device__ __forceinline__ void scores(f32x4 (&x)[MT][2], const Rows<T, D, MT>& w, const u32x4 (&k)[2][D / 32], const Place& t,
                                       int k0, int g) {
  typedef typename Mat<T>::x8 x8;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int seen = (t.ok[h] ? TAIL ? w.lim[mt] : 0x7fffffff : 0) - (k0 + 16 * h + 4 * g);
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) s = Mat<T>::mul(__builtin_bit_cast(x8, k[h][c]), w.q[mt][c], s);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[mt][h][j] = (TAIL ? j < seen : t.ok[h]) ? s[j] : -INFINITY;
    }
  }
}

// Scores to weights, against the running maximum.  Scores are scaled behind the difference: a maximum that is itself scaled
// and rounded is off by half a step of its own, which from scores of 2^31 on is more than the exponential's range.
template <typename T, int D, int MT>
__device__ __forceinline__ void weights(typename Mat<T>::x8 (&hi)[MT], typename Mat<T>::x8 (&lo)[MT], Rows<T, D, MT>& w,
                                        const f32x4 (&x)[MT][2], float scale2) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(x[mt][0][j], x[mt][1][j]));
    if (__any(top > w.m[mt])) {                              // rare once the largest scores have been seen
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float m = fmaxf(w.m[mt], top);
      const float a = __builtin_amdgcn_exp2f((w.m[mt] - m) * scale2);
      w.m[mt] = m;
      w.l[mt] *= a;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) w.o[mt][i][j] *= a;
    }
    float sum = 0.f;
    u32x4 h4, l4;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int h = c >> 1, j = 2 * (c & 1);
      const float e0 = __builtin_amdgcn_exp2f((x[mt][h][j] - w.m[mt]) * scale2 + Mat<T>::UP);
      const float e1 = __builtin_amdgcn_exp2f((x[mt][h][j + 1] - w.m[mt]) * scale2 + Mat<T>::UP);
      sum += e0 + e1;
      uint32_t a, b;
      Mat<T>::split(e0, e1, a, b);
      h4[c] = a;
      l4[c] = b;
    }
    hi[mt] = __builtin_bit_cast(typename Mat<T>::x8, h4);
    lo[mt] = __builtin_bit_cast(typename Mat<T>::x8, l4);
    w.l[mt] += sum;                                          // this lane's keys; the four lane groups join at the end
  }
}

// Weights times values into the rows' sums.
template <typename T, int D, int MT, bool TAIL>
__device__ __forceinline__ void add_values(Rows<T, D, MT>& w, uint32_t (&v)[8][D / 32], const typename Mat<T>::x8 (&hi)[MT],
                                           const typename Mat<T>::x8 (&lo)[MT], const Place& t, int k0,
                                           int limit_all, int limit, int g, bool& odd) {
  typedef typename Mat<T>::x8 x8;
  if (TAIL) {
    // Rows of later tokens see keys that rows of earlier ones do not.  A product of a hidden key's weight, 0, and a value
    // that is no finite number would be NaN, so such values leave the product here, and the sums are taken once more at the end.
    constexpr uint32_t EXP = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int key = k0 + 16 * (s >> 2) + 4 * g + (s & 3);
      const bool none = key >= limit, some = key >= limit_all;
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

// The wave's m, l and o once more, element by element, for data the products above do not serve: a value that is no
// finite number at a position that some rows see and others do not (0 x NaN), or an infinite one (hi and lo weights of both
// signs).  Scores are summed in another order here, and where they are large that moves a weight by more than a rounding, so
// maximum and sum are taken from these scores too.
template <typename T, int D, int MT, int TK>
__device__ __forceinline__ void add_values_again(Rows<T, D, MT>& w, const PagedAttArgs& p, const_i32 row, int b, int hk, int row0,
                                                 int R, int G, int first, int limit, int r, int g) {
  typedef typename Mat<T>::x8 x8;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    w.m[mt] = ROW_NONE;
    w.l[mt] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) w.o[mt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 1
  for (int k0 = first; k0 < limit; k0 += TK) {
#pragma unroll 1
    for (int key = k0; key < min(k0 + 32, limit); ++key) {
      const int pi = key / p.page, pid = row[pi];
      if (pid < 0 || pid >= p.pages) continue;
      const long long slot = key - pi * p.page;
      const T* kr = (const T*)((const char*)p.kp + pid * p.k_ps + slot * p.k_ss + hk * p.k_hs);
      const T* vr = (const T*)((const char*)p.vp + pid * p.v_ps + slot * p.v_ss + hk * p.v_hs) + D / 4 * g;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int at = row0 + 16 * mt + r, i = at / G, h = hk * G + at - i * G;
        if (at >= R || key >= w.lim[mt]) continue;
        const T* qr = (const T*)p.q + b * p.q_bs + i * p.q_ns + h * p.q_hs;
        float x = 0.f;
#pragma unroll 1
        for (int d = 0; d < D; d += 8) {
          const x8 a = *reinterpret_cast<const x8*>(qr + d), c = *reinterpret_cast<const x8*>(kr + d);
#pragma unroll
          for (int j = 0; j < 8; ++j) x += (float)a[j] * (float)c[j];
        }
        x = p.flip ? -x : x;
        if (x > w.m[mt]) {
          const float a = __builtin_amdgcn_exp2f((w.m[mt] - x) * p.scale2);
          w.m[mt] = x;
          w.l[mt] *= a;
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) w.o[mt][i][j] *= a;
        }
        const float e = __builtin_amdgcn_exp2f((x - w.m[mt]) * p.scale2 + Mat<T>::UP);
        if (g == 0) w.l[mt] += e;                            // the lane groups' sums are added up; here each has all keys
#pragma unroll
        for (int d = 0; d < D / 4; d += 8) {                 // the lane's sums: dimensions D / 4 g .. of its query
          const x8 v = *reinterpret_cast<const x8*>(vr + d);
#pragma unroll
          for (int j = 0; j < 8; ++j) w.o[mt][(d + j) % (D / 16)][(d + j) / (D / 16)] += e * (float)v[j];
        }
      }
    }
  }
}

// Tiles of a sequence that keeps so many tokens (at least one: an empty sequence's rows are written, too).
template <int TK>
__device__ __forceinline__ int tiles_of(const PagedAttArgs& p, int kept) {
  const int cap = p.width * p.page;
  const int limit = kept < 0 || p.pages == 0 ? 0 : min(min(kept, cap) + (p.causal ? p.n : 0), cap);
  return max(1, (limit + TK - 1) / TK);
}

// Sum over the lanes up to and with this one: shifts inside rows of 16 lanes, then the last lanes of rows to the rows behind.
__device__ __forceinline__ int wave_scan_i32(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) {
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x111, 0xf, 0xf, false));
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x112, 0xf, 0xf, false));
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x114, 0xf, 0xf, false));
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x118, 0xf, 0xf, false));
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x142, 0xa, 0xf, false));
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x143, 0xc, 0xf, false));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// How tiles are dealt out.  A problem is a sequence's key head and group of rows, H of them per sequence.  Parts have `each`
// tiles, a problem's last one less; they are numbered problem after problem.  each is at least max(least, all tiles / share), so
// there are at most share + problems parts.  Short last parts may make them more than the `share` workgroups that are resident
// at once, and a further round is not free: one workgroup alone takes 0.1 of the time that it takes among all of them, where
// a row tile has few registers and the memory is the bound, 0.7 where it has many (more than 16 rows).  Then, of 64 lengths
// from the least one to twice that, a lane each, the one that ends first by that reckoning is taken.  12 sequences x 8 heads
// of 6000 keys, 20 rows: 86 us with the least length, 67 so; 40 x 8 heads, one row of 64: 118 and 97.
// mine: tiles of sequence `lane`, of the first 64, 0 where there is none.
template <int TK>
__device__ __forceinline__ int tiles_each(const PagedAttArgs& p, int H, int lane, int mine) {
  int sum = mine;
  for (int b = lane + 64; b < p.B; b += 64) sum += tiles_of<TK>(p, p.lens[b]);
  const int total = __builtin_amdgcn_readlane(wave_scan_i32(sum), 63) * H;
  if (total <= p.share) return p.least;
  const int least = max(p.least, (total + p.share - 1) / p.share);
  if (p.B > 64 || p.B * H >= p.share) return least;          // more rounds than one in any case
  if (__builtin_amdgcn_readlane(wave_scan_i32((mine + least - 1) / least), 63) * H <= p.share) return least;
  const uint32_t each = least + lane * (1 + (least >> 6)), magic = 0xffffffffu / each + 1;      // umulhi(t, magic): t / each, or near it
  uint32_t parts = 0;
  for (int b = 0; b < p.B; b += 8)
#pragma unroll
    for (int x = 0; x < 8; ++x) parts += __umulhi(__builtin_amdgcn_readlane(mine, b + x) + each - 1, magic);
  const int over = (int)parts * H - p.share, few = 31 - __clz(least | 1 << 13) - 13;
  const uint32_t more = over <= 0 ? 0 : max((uint32_t)over * 256u / (uint32_t)p.share, p.rows > 16 ? 180u : 26u);
  const int best = (int)(wave_min_u32((each >> few) * (256u + more) << 6 | lane) & 63u);
  return __builtin_amdgcn_readlane((int)each, best);
}

template <typename T, int D, int MT>
__global__ __launch_bounds__(256, MT == 1 ? 3 : MT == 2 ? 2 : 1) void paged_attention_kernel(const PagedAttArgs p) {
  typedef typename Mat<T>::x8 x8;
  constexpr int TK = 128;                                    // keys of a tile: 32 for each wave
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ float s_o[4][16][D + 4];                        // + 4: lanes of one group write 16 rows at once
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int G = p.Hq / p.Hkv, R = p.n * G, H = p.Hkv * p.groups;
  // groups of rows that read the same keys, on one die: 64 rows over 100000 keys 105 us, dealt out in turn 132; 128 rows, 8 x
  // 9000 72 and 102; 40 rows, 96 heads x 1500 27.1 and 29.5
  const int cap = p.width * p.page, me = dlamd_xcd_neighbours(blockIdx.x, p.groups, gridDim.x);

  // which problem and which of its tiles
  int b, head, kept, tile = 0, tiles = 0x7fffffff;
  bool whole = true;
  if (p.share == 0) {
    b = me / H;
    head = me - b * H;                                       // groups of one key head side by side
    b = __builtin_amdgcn_readfirstlane(b);
    kept = ((const_i32)p.lens)[b];
  } else {
    int mine = lane < p.B ? p.lens[lane] : 0;
    const int t0 = lane < p.B ? tiles_of<TK>(p, mine) : 0;
    const int each = tiles_each<TK>(p, H, lane, t0);
    if (me == 0 && threadIdx.x == 0) reinterpret_cast<int*>(p.part)[D + 2] = each;    // for the join
    int begin = 0, src = -1, upto = 0, parts = 0;
    b = 0;
    for (; b < p.B; b += 64) {                               // the sequence of part `me`, 64 of them at a time
      if (b) mine = b + lane < p.B ? p.lens[b + lane] : 0;
      const int t = b == 0 ? t0 : b + lane < p.B ? tiles_of<TK>(p, mine) : 0;
      parts = (t + each - 1) / each;
      upto = begin + wave_scan_i32(parts * H);
      const unsigned long long past = __ballot(upto > me);
      if (past) {
        src = __ffsll(past) - 1;
        break;
      }
      begin = __builtin_amdgcn_readlane(upto, 63);
    }
    if (src < 0) return;                                     // fewer parts than workgroups
    b += src;
    kept = __builtin_amdgcn_readlane(mine, src);
    parts = __builtin_amdgcn_readlane(parts, src);
    const int in = me - (__builtin_amdgcn_readlane(upto, src) - parts * H);
    const int unit = in / p.groups;                          // key head after key head, part after part, group after group
    const int h = unit / parts;
    head = h * p.groups + in - unit * p.groups;
    tile = (unit - h * parts) * each;
    tiles = each;
    whole = parts == 1;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  head = __builtin_amdgcn_readfirstlane(head);
  tile = __builtin_amdgcn_readfirstlane(tile);

  // the first pages are asked for together with the length, not after it
  const const_i32 row = (const_i32)p.table + b * p.t_bs;
  const int kb = tile * TK;
  int k0 = kb + 32 * wave;
  const int first0 = page_of(p, row, k0), first1 = page_of(p, row, k0 + 16);
  int pid0 = page_of(p, row, k0 + TK), pid1 = page_of(p, row, k0 + TK + 16);
  const int hk = head / p.groups, row0 = (head - hk * p.groups) * p.rows;
  Rows<T, D, MT> w;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + r, i = row / G, h = hk * G + row - i * G;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      u32x4 t = {0u, 0u, 0u, 0u};
      if (row < R) t = *reinterpret_cast<const u32x4*>((const T*)p.q + b * p.q_bs + i * p.q_ns + h * p.q_hs + 32 * c + 8 * g);
      w.q[mt][c] = __builtin_bit_cast(x8, t ^ p.flip);
    }
  }
  const int base = kept < 0 || p.pages == 0 ? 0 : min(kept, cap), more = kept >= 0 && p.pages > 0 && p.causal;
  // limits of the first and last row
  const int rl = min(row0 + 16 * MT, R) - 1;
  const int limit_all = min(base + (more ? row0 / G + 1 : 0), cap);
  const int limit = (int)min((long long)min(base + (more ? rl / G + 1 : 0), cap), ((long long)tile + tiles) * TK);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = row0 + 16 * mt + r;
    w.lim[mt] = row < R ? min(min(base + (more ? row / G + 1 : 0), cap), limit) : 0;
    w.m[mt] = ROW_NONE;
    w.l[mt] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) w.o[mt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // The next tile's keys are fetched into the registers of this one's as soon as the scores have been taken, its values
  // after the products: at any time a wave has most of a tile in flight, and three waves fit a SIMD.
  const global_p kh = (global_p)p.kp + hk * p.k_hs, vh = (global_p)p.vp + hk * p.v_hs;
  bool odd = false;
  if (k0 < limit) {
    u32x4 k[2][D / 32];
    uint32_t v[8][D / 32];
    Place pl;
    x8 hi[MT], lo[MT];
    f32x4 x[MT][2];
    find_tile(pl, p, kh, vh, first0, first1, k0, limit);
    load_k<D, true>(k, pl, r, g);
    load_v<D, true>(v, pl, r, g);
    // All tiles but a wave's last end more than 96 keys before the limit, and the first row's limit is at most 63 keys before
    // that: every row sees them.  No load here has a condition: where a path with loads meets one without, the compiler can
    // only wait for all of them.
    for (; k0 + TK < limit; k0 += TK) {
      scores<T, D, MT, false>(x, w, k, pl, k0, g);
      Place next;
      find_tile(next, p, kh, vh, pid0, pid1, k0 + TK, limit);
      load_k<D, true>(k, next, r, g);
      pid0 = page_of(p, row, k0 + 2 * TK);
      pid1 = page_of(p, row, k0 + 2 * TK + 16);
      weights<T, D, MT>(hi, lo, w, x, p.scale2);
      add_values<T, D, MT, false>(w, v, hi, lo, pl, k0, limit_all, limit, g, odd);
      load_v<D, true>(v, next, r, g);
      pl = next;
    }
    scores<T, D, MT, true>(x, w, k, pl, k0, g);
    weights<T, D, MT>(hi, lo, w, x, p.scale2);
    add_values<T, D, MT, true>(w, v, hi, lo, pl, k0, limit_all, limit, g, odd);
  }
  // Only rows that are written count: a row of zeros that fills a tile up is NaN from any key with an infinite component.
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) nan |= w.o[mt][i][j] != w.o[mt][i][j];
    odd |= nan && r < min(p.rows, R - row0) - 16 * mt;
  }
  if (__any(odd)) add_values_again<T, D, MT, TK>(w, p, row, b, hk, row0, R, G, kb + 32 * wave, limit, r, g);
  float* part = p.part + (long long)me * p.rows * (D + 4);
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
    // a thread: D / 16 dimensions of a row
    const int rr = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16), in = 16 * mt + rr, row = row0 + in;
    if (in < p.rows && row < R) {
      const float m = fmaxf(fmaxf(s_m[0][rr], s_m[1][rr]), fmaxf(s_m[2][rr], s_m[3][rr]));
      float f[4], sum = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        f[x] = __builtin_amdgcn_exp2f((s_m[x][rr] - m) * p.scale2);
        sum += f[x] * s_l[x][rr];
      }
      float o[D / 16];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        o[d] = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[d] += f[x] * s_o[x][rr][d0 + d];
      }
      if (whole) {
        const int i = row / G, h = hk * G + row - i * G;
        const long long to = ((long long)b * p.n + i) * p.Hq + h;
        const float inv = 1.f / sum;
        T t[D / 16];
#pragma unroll
        for (int d = 0; d < D / 16; ++d) t[d] = (T)(sum == 0.f ? 0.f : o[d] * inv);   // sum is NaN where a score is
        T* dst = (T*)p.o + to * D + d0;
#pragma unroll
        for (int d = 0; d < D / 16; d += 4) *reinterpret_cast<u32x2*>(dst + d) = *reinterpret_cast<u32x2*>(t + d);
        if (p.lse && d0 == 0) p.lse[to] = sum == 0.f ? -INFINITY : (m * p.scale2 + __log2f(sum * Mat<T>::DOWN)) * LN2;
      } else {
        float* dst = part + in * (D + 4);
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

// One workgroup per row: joins the parts of its sequence.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(const PagedAttArgs p) {
  constexpr int TK = 128;
  constexpr int TD = D / 4, SL = 256 / TD;                   // threads per part (4 dimensions each), parts side by side
  __shared__ float s_o[SL][D];
  __shared__ float s_l[SL], s_m[SL];
  const long long to = blockIdx.x;
  const int h = (int)(to % p.Hq), i = (int)((to / p.Hq) % p.n), b = (int)(to / ((long long)p.Hq * p.n));
  const int G = p.Hq / p.Hkv, H = p.Hkv * p.groups, hk = h / G;
  const int row = i * G + h - hk * G, group = row / p.rows, in = row - group * p.rows;
  const int lane = threadIdx.x & 63;
  const int own = ((const_i32)p.lens)[b];
  const int each = reinterpret_cast<const int*>(p.part)[D + 2];
  const int parts = (tiles_of<TK>(p, own) + each - 1) / each;
  if (parts == 1) return;                                    // written already
  int before = 0;                                            // parts of the sequences before this one
  for (int x = lane; x < b; x += 64) before += (tiles_of<TK>(p, p.lens[x]) + each - 1) / each;
  const int lo = __builtin_amdgcn_readlane(wave_scan_i32(before), 63) * H + hk * parts * p.groups + group;
  const int d = (threadIdx.x % TD) * 4, sl = threadIdx.x / TD;
  const float* src = p.part + (long long)in * (D + 4);
  float m = ROW_NONE, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = sl; s < parts; s += SL) {
    const float* q = src + (long long)(lo + s * p.groups) * p.rows * (D + 4);
    const float ms = q[D], ls = q[D + 1], mn = fmaxf(m, ms);
    const f32x4 os = *reinterpret_cast<const f32x4*>(q + d);
    const float a = __builtin_amdgcn_exp2f((m - mn) * p.scale2), c = __builtin_amdgcn_exp2f((ms - mn) * p.scale2);
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
    float top = ROW_NONE, sum2 = 0.f, v = 0.f;
#pragma unroll
    for (int x = 0; x < SL; ++x) top = fmaxf(top, s_m[x]);
#pragma unroll
    for (int x = 0; x < SL; ++x) {
      const float f = __builtin_amdgcn_exp2f((s_m[x] - top) * p.scale2);
      sum2 += f * s_l[x];
      v += f * s_o[x][threadIdx.x];
    }
    ((T*)p.o)[to * D + threadIdx.x] = (T)(sum2 == 0.f ? 0.f : v / sum2);
    if (p.lse && threadIdx.x == 0) p.lse[to] = sum2 == 0.f ? -INFINITY : (top * p.scale2 + __log2f(sum2 * Mat<T>::DOWN)) * LN2;
  }
}

template <typename T, int D, int MT>
static void launch(const PagedAttArgs& a, hipStream_t stream) {
  const unsigned grid = a.share + a.B * a.Hkv * a.groups;
  hipLaunchKernelGGL((paged_attention_kernel<T, D, MT>), dim3(grid), dim3(256), 0, stream, a);
  if (a.share)
    hipLaunchKernelGGL((paged_attention_join_kernel<T, D>), dim3((unsigned)(a.B * a.n * a.Hq)), dim3(256), 0, stream, a);
}
template <typename T, int D>
static void launch_rows(const PagedAttArgs& a, int rows, hipStream_t stream) {
  if (rows <= 16) launch<T, D, 1>(a, stream);
  else if (rows <= 32) launch<T, D, 2>(a, stream);
  else launch<T, D, 3>(a, stream);
}

// q: [B, n, Hq, D] (strides given), o: [B, n, Hq, D] contiguous, lse: [B, n, Hq] or null.  dtype: 0 bf16, 1 fp16.
// groups: the n x Hq / Hkv rows that read one key head in so many groups, of at most 48.
// share: 0 (a workgroup per sequence, key head and group of rows) or workgroups to deal all tiles out to, in parts of at least
// `least` tiles; part: [share + problems][rows of a problem][D + 4] floats where share > 0.
extern "C" int dlamd_paged_attention(const void* q, long long q_bs, long long q_ns, long long q_hs, const void* kp,
                                     long long kp_ps, long long kp_ss, long long kp_hs, const void* vp, long long vp_ps,
                                     long long vp_ss, long long vp_hs, const void* table, long long t_bs,
                                     const void* lens, void* o, void* lse, void* part, long long part_floats,
                                     int groups, int share, int least, int B, int n,
                                     int Hq, int Hkv, int D, int page, int width, int pages, int causal, float scale,
                                     int dtype, hipStream_t stream) {
  if (B <= 0 || n <= 0 || Hq <= 0) return 0;
  if (Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128)) return -1;
  if (page <= 0 || page % 16 != 0 || width < 0 || pages < 0) return -2;
  if ((q_bs | q_ns | q_hs | kp_ps | kp_ss | kp_hs | vp_ps | vp_ss | vp_hs) % 8 != 0) return -3;
  if (((uintptr_t)q | (uintptr_t)kp | (uintptr_t)vp | (uintptr_t)o) & 15) return -4;
  // a lane's offset inside 16 slots is a 24-bit product, a slot's inside its page 32 bits
  const long long sl[2] = {kp_ss * 2, vp_ss * 2};
  if (sl[0] < 0 || sl[1] < 0 || sl[0] >= (1 << 24) || sl[1] >= (1 << 24) || page * sl[0] > 0x7fffffff || page * sl[1] > 0x7fffffff)
    return -11;
  // positions are 32-bit; the page of a position is a multiplication, exact while units * (page / 16) < 2^32
  if ((long long)width * page > 0x7ff00000LL || (long long)width * (page / 16) * (page / 16) >= (1LL << 32)) return -5;
  if (dtype != 0 && dtype != 1) return -6;
  if (share < 0 || share > (1 << 20) || (share > 0 && (least < 1 || !part || ((uintptr_t)part & 15)))) return -7;
  if ((long long)n * Hq > 0x7fffffffLL || (share > 0 && (long long)n * Hq >= (1LL << 24) / B)) return -9;   // the join: a workgroup per row
  const int R = n * (Hq / Hkv);
  if (groups < 1 || groups > R || (R + groups - 1) / groups > 48) return -8;
  const int rows = (R + groups - 1) / groups;
  if (share > 0 && part_floats < ((long long)share + (long long)B * Hkv * groups) * rows * (D + 4)) return -12;
  // problems, parts and tiles are counted in 32 bits, the launch in 2^24 workgroups
  if ((long long)B * Hkv * groups + share >= (1LL << 24)) return -10;
  if (((long long)B * Hkv * groups + share) * ((long long)width * page / 64 + 2) > 0x7fffffffLL) return -10;
  if (width == 0) {                                          // no table to read: one entry of anything, and no pages
    table = lens;
    t_bs = 0;
    width = 1;
    pages = 0;
  }
  const uint32_t units = (uint32_t)(page / 16);
  const uint32_t magic = units == 1 ? 0u : (uint32_t)((0x100000000ULL + units - 1) / units);
  PagedAttArgs a{q, kp, vp, o, (float*)lse, (float*)part, (const int*)table, (const int*)lens, q_bs, q_ns, q_hs,
                 kp_ps * 2, kp_hs * 2, vp_ps * 2, vp_hs * 2, t_bs, (int)sl[0], (int)sl[1], B, n, Hq, Hkv, page, width, pages, causal,
                 groups, rows, share, least, magic, fmaxf(fabsf(scale) * 1.4426950408889634f, 1.17549435e-38f), scale < 0.f ? 0x80008000u : 0u};
  if (dtype == 0 && D == 64) launch_rows<bf16_t, 64>(a, rows, stream);
  if (dtype == 0 && D == 128) launch_rows<bf16_t, 128>(a, rows, stream);
  if (dtype == 1 && D == 64) launch_rows<f16_t, 64>(a, rows, stream);
  if (dtype == 1 && D == 128) launch_rows<f16_t, 128>(a, rows, stream);
  return DLAMD_CHECK_LAUNCH();
}
