// C entries of the decode-step operators' kernels, as their host side (csrc/bind/decode_ops.cpp) calls them.  Included by both,
// so that a definition and its caller cannot disagree.  Return 0, or a negative code where the contract on sizes, strides,
// alignment or workspaces does not hold (nothing is launched then).  Strides are in elements; dtype 0 bf16, 1 fp16, 2 fp32.
#pragma once

struct ihipStream_t;

extern "C" {
int dlamd_paged_append(const void* k, long long k_ts, long long k_hs, const void* v, long long v_ts, long long v_hs, const void* q,
                       long long q_ts, long long q_hs, void* qo, void* kp, long long kp_ps, long long kp_ss, long long kp_hs, void* vp,
                       long long vp_ps, long long vp_ss, long long vp_hs, const void* table, long long t_bs, const void* lens,
                       const void* starts, const void* cs, const void* sn, int B, int T, int Hq, int Hkv, int D, int rot, int page,
                       int width, int pages, int interleaved, int dtype, ihipStream_t* stream);
int dlamd_paged_attention(const void* q, long long q_bs, long long q_ns, long long q_hs, const void* kp, long long kp_ps,
                          long long kp_ss, long long kp_hs, const void* vp, long long vp_ps, long long vp_ss, long long vp_hs,
                          const void* table, long long t_bs, const void* lens, void* o, void* lse, void* part, long long part_floats,
                          int groups, int share, int least, int B, int n, int Hq, int Hkv, int D, int page, int width, int pages, int causal,
                          float scale, int dtype, ihipStream_t* stream);
int dlamd_verify_draft(const void* draft, long long d_bs, const void* p, long long p_bs, long long p_ns, const void* q, long long q_bs,
                       long long q_ns, const void* u, long long u_bs, const void* counts, void* tokens, void* accepted, void* sums,
                       long long sums_doubles, int pieces, int B, int n, int V, int pad, int dtype, ihipStream_t* stream);
int dlamd_int4_linear(const void* x, long long x_rs, const void* w, const void* scale, const void* zero, const void* bias,
                      const void* res, long long res_rs, void* y, int M, int N, int K, int G, int act, int dtype, int sdtype, int tiles,
                      int nw, int kw, int kz, void* part, long long part_floats, ihipStream_t* stream);
}
