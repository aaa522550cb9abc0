// The host side of the decode-step operators (ops/paged.py, ops/int4.py, ops/draft.py) on device tensors: argument checks,
// outputs and workspaces from PyTorch's allocator, the launch.
//
// A decode step is made of calls whose kernels take 3 to 10 us, so the host has to issue one in less than that.  In Python a
// call cost 8.7 us (3.4 us of it the launch itself, 2.8 us two allocations, the rest reading sizes, strides and addresses one by
// one); here 5 us.  The kernels are the plain C entries of libdlamd_kernels.so, whose addresses Python hands over once (init).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../kernels/decode_abi.h"

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

namespace {

typedef long long ll;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct Failed : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void need(bool ok, const char* why) {
  if (!ok) throw Refused(why);
}
void launched(int rc, const char* name) {
  if (rc != 0)
    throw Failed(std::string(name) + " failed with code " + std::to_string(rc) + " (host-side shape contract or launch error)");
}

decltype(&dlamd_paged_append) k_append;
decltype(&dlamd_paged_attention) k_attention;
decltype(&dlamd_verify_draft) k_verify;
decltype(&dlamd_int4_linear) k_int4;
PyObject* k_error = nullptr;                                 // the framework's KernelLibraryError

// ------------------------------------------------------------------------------------------ arguments
struct Maybe {
  const at::Tensor* t = nullptr;
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor* operator->() const { return t; }
  const void* ptr() const { return t ? t->data_ptr() : nullptr; }
};
Maybe maybe(PyObject* o) {
  if (o == Py_None) return {};
  need(THPVariable_Check(o), "a tensor or None is expected");
  return {&THPVariable_Unpack(o)};
}
const at::Tensor& tensor(PyObject* o) {
  need(THPVariable_Check(o), "a tensor is expected");
  return THPVariable_Unpack(o);
}
ll number(PyObject* o) {
  const ll v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refused("a whole number is expected");
  }
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    throw Refused("a truth value is expected");
  }
  return v == 1;
}

// Device of the call, made current for the launch, and its current stream as Python knows it.
struct Where {
  c10::DeviceGuard guard;
  ihipStream_t* stream;
  Where(const at::Tensor& t, PyObject* s) : guard(t.device()), stream((ihipStream_t*)(intptr_t)number(s)) {}
};
void same_device(const c10::Device& d, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts) need(!t || t->device() == d, "all tensors live on one device");
}

// The operators have no derivatives: a result that silently carried no gradient would train nothing, one without its tangent
// would be a constant in forward mode (which torch.no_grad() leaves on).
void no_gradient(std::initializer_list<const at::Tensor*> ts) {
  const bool backward = c10::GradMode::is_enabled();
  const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0);
  for (const at::Tensor* t : ts) {
    need(!backward || !t || !t->requires_grad(), "the operator has no gradient: call it under torch.no_grad() or on detached tensors");
    need(!forward || !t || !t->_fw_grad(0).defined(), "the operator has no forward-mode derivative: call it on detached tensors");
  }
}

// A dimension of one element has whatever stride: none is asked of it, and none is passed on.
bool packed(const at::Tensor& t, int d) { return t.size(d) < 2 || t.stride(d) == 1; }
ll step(const at::Tensor& t, int d) { return t.size(d) < 2 ? 0 : t.stride(d); }

int half_type(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : -1; }

void check_cache(const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& table, const at::Tensor& lens) {
  need(kp.dim() == 4 && vp.sizes() == kp.sizes(), "k_pages and v_pages are [pages, page, kv_heads, D] of one shape");
  need(half_type(kp.scalar_type()) >= 0 && vp.scalar_type() == kp.scalar_type(), "the cache is bf16 or fp16");
  need(table.dim() == 2 && table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == table.size(0),
       "table is int32 [B, width], lens int32 [B]");
  need(packed(kp, 3) && packed(vp, 3) && packed(table, 1) && packed(lens, 0),
       "the last dimensions of the cache, of table and of lens have to be contiguous");
}
int as_int(int64_t v) {
  need(v >= 0 && v <= 0x7fffffff, "a size beyond 31 bits");
  return (int)v;
}

// ------------------------------------------------------------------------------------------ append
// (k, v, k_pages, v_pages, table, lens, q, cos, sin, starts, interleaved, stream) -> q rotated or None
PyObject* append(PyObject* const* a) {
  const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &kp = tensor(a[2]), &vp = tensor(a[3]), &table = tensor(a[4]), &lens = tensor(a[5]);
  const Maybe q = maybe(a[6]), cos = maybe(a[7]), sin = maybe(a[8]), starts = maybe(a[9]);
  check_cache(kp, vp, table, lens);
  const int64_t B = table.size(0), width = table.size(1), page = kp.size(1), hkv = kp.size(2), D = kp.size(3);
  need(k.dim() == 3 && k.sizes() == v.sizes() && k.size(1) == hkv && k.size(2) == D, "k and v are [T, kv_heads, D] with the cache's heads and D");
  const int64_t T = k.size(0);
  const at::ScalarType dt = kp.scalar_type();
  need(k.scalar_type() == dt && v.scalar_type() == dt && packed(k, 2) && packed(v, 2),
       "k and v have the cache's type and a contiguous last dimension");
  need(D % 8 == 0 && hkv > 0, "D is a multiple of 8, the cache has heads");
  no_gradient({&k, &v, &kp, &vp, q.t, cos.t, sin.t});
  same_device(k.device(), {&v, &kp, &vp, &table, &lens, q.t, cos.t, sin.t, starts.t});
  if (q)
    need(q->dim() == 3 && q->size(0) == T && q->size(1) > 0 && q->size(2) == D && q->scalar_type() == dt && packed(*q.t, 2),
         "q is [T, heads, D] of the cache's type and device with a contiguous last dimension");
  need((bool)cos == (bool)sin, "cos and sin come together");
  int64_t rot = 0;
  if (cos) {
    need(cos->dim() == 2 && cos->sizes() == sin->sizes(), "cos and sin are [P, rot / 2] with P >= width * page, rot <= D and rot % 16 == 0");
    rot = 2 * cos->size(1);
    need(cos->size(0) >= width * page && rot <= D && rot % 16 == 0, "cos and sin are [P, rot / 2] with P >= width * page, rot <= D and rot % 16 == 0");
    need(cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat && cos->is_contiguous() && sin->is_contiguous(),
         "cos and sin are contiguous fp32");
  }
  if (starts)
    need(starts->scalar_type() == at::kInt && starts->dim() == 1 && starts->size(0) == B + 1 && packed(*starts.t, 0),
         "starts is int32 [B + 1] on the cache's device");
  else
    need((B ? T % B : T) == 0, "without starts every sequence has the same number of new tokens");
  const Where w(k, a[11]);
  at::Tensor qo;
  if (q) qo = B && width ? at::empty({T, q->size(1), D}, q->options()) : at::zeros({T, q->size(1), D}, q->options());
  launched(k_append(k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(), step(v, 0), step(v, 1), q.ptr(), q ? step(*q.t, 0) : 0,
                    q ? step(*q.t, 1) : 0, q ? qo.data_ptr() : nullptr, kp.data_ptr(), step(kp, 0), step(kp, 1), step(kp, 2), vp.data_ptr(),
                    step(vp, 0), step(vp, 1), step(vp, 2), table.data_ptr(), step(table, 0), lens.data_ptr(), starts.ptr(), cos.ptr(),
                    sin.ptr(), as_int(B), as_int(T), q ? as_int(q->size(1)) : 0, as_int(hkv), as_int(D), (int)rot, as_int(page), as_int(width),
                    as_int(kp.size(0)), truth(a[10]), half_type(dt), w.stream),
           "dlamd_paged_append");
  if (!q) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(qo));
}

// ------------------------------------------------------------------------------------------ attention
struct Deal {
  int64_t share, least;
};
// How a call's tiles of keys are dealt out: {0, 0}, a workgroup per problem (sequence, key head, group of rows), or workgroups to
// deal all tiles out to and the least tiles of a part.
//   * Parts cost a join, some 6 us, as long as a workgroup takes for 6 or 7 tiles of 128 keys.  So a workgroup per problem,
//     unless parts spare each workgroup more than that: 96 heads x 1024 keys 10.1 us, in parts 12.6; 160 x 155 keys, 24 rows,
//     9.1 and 17.9; 320 x 2048, 40 rows, 53 and 67; but 8 x 2048 keys 14.5 and 8.4, 96 x 6000 57 and 35.
//   * Only the bound is known here.  Beyond 4096 keys lengths may differ much, which parts even out: 320 x up to 6000 keys, 20
//     rows, 57.4 us one workgroup each, 32.8 in parts (all of one length: 135 and 144).
//   * Otherwise as many workgroups as are resident at once by their registers, 3 per compute unit for D 128, 4 for D 64:
//     8 x 16384 keys, 8 heads of 128: 101 us with 768, 103 with 256.
//   * A part's (m, l, o) costs rows x D floats written and read: beyond 16 rows one workgroup per compute unit.  2 x 16384 keys,
//     64 rows: 26.6 us with 256, 29.7 with 512; 12 ragged caches of up to 8009 keys, 40 rows: 26 and 34.
Deal deal_out(int64_t problems, int64_t rows, int64_t bound, int64_t D) {
  const int64_t share = rows > 16 ? 256 : D == 64 ? 1024 : 768, resident = rows > 32 ? 256 : rows > 16 ? 512 : share;
  if (bound <= 4096) {
    const int64_t tiles = (bound + 127) / 128, whole = (problems + resident - 1) / resident * tiles;
    if (whole - (problems * tiles + share - 1) / share < 7) return {0, 0};
  }
  return {share, 1};
}

// The rows (new tokens x query heads) that read one key head, in groups of up to 48, three tiles of 16.  Three tiles in a wave
// fetch a key once, but leave one workgroup per compute unit; two groups of two tiles side by side have two, which is worth
// more while the keys are few: 8 heads x 3000 keys, 40 rows, 17.3 us as one group and 15.0 as two, 96 x 1500 33.1 and 27.3, 16 x
// 6000 23.2 and 22.6; but 8 x 24000 32.5 and 33.8, 96 x 6000 72 and 88, 320 x 2048 with heads of 64 53 and 62.  More rows:
// groups of up to 32 (2 x 16384 keys, 64 rows: 26.5 us, in one wave 30).
int64_t row_groups(int64_t rows, int64_t heads, int64_t bound) {
  if (rows <= 32) return 1;
  if (rows > 48) return (rows + 31) / 32;
  return (bound <= 2048 && heads < 256) || heads * ((bound + 127) / 128) <= 1000 ? 2 : 1;
}

// (q, k_pages, v_pages, table, lens, scale or None, causal, max_len or None, return_lse, share or None, least, stream)
PyObject* attention(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0]), &kp = tensor(a[1]), &vp = tensor(a[2]), &table = tensor(a[3]), &lens = tensor(a[4]);
  check_cache(kp, vp, table, lens);
  need(q.dim() == 4 && q.scalar_type() == kp.scalar_type() && packed(q, 3),
       "q is [B, n, heads, D] of the cache's type with a contiguous last dimension");
  const int64_t B = q.size(0), n = q.size(1), hq = q.size(2), D = q.size(3), page = kp.size(1), hkv = kp.size(2), width = table.size(1);
  need(table.size(0) == B && kp.size(3) == D && hkv > 0 && hq % hkv == 0,
       "q, table and cache disagree: one table row per sequence, D alike, heads a multiple of kv_heads");
  need(page > 0 && page % 16 == 0 && (D == 64 || D == 128), "page is a multiple of 16, D is 64 or 128");
  no_gradient({&q, &kp, &vp});
  same_device(q.device(), {&kp, &vp, &table, &lens});
  double scale = 1.0 / std::sqrt((double)D);
  if (a[5] != Py_None) {
    scale = PyFloat_AsDouble(a[5]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      throw Refused("scale is a number");
    }
    need(std::fabs(scale) <= 2e38, "scale is a number of at most 2e38");        // its product with log2(e) fits 32 bits
  }
  int64_t bound = width * page;
  if (a[7] != Py_None) bound = std::min<int64_t>(bound, number(a[7]));
  const int64_t all = n * (hq / hkv), groups = row_groups(all, B * hkv, bound), rows = (all + groups - 1) / groups;
  const int64_t problems = B * hkv * groups;
  Deal d = a[9] == Py_None ? deal_out(problems, rows, bound, D) : Deal{number(a[9]), number(a[10])};
  if (n * hq >= (int64_t)(1 << 24) / std::max<int64_t>(B, 1)) d = {0, 0};     // the join's launch ends there, and the card is full
  const Where w(q, a[11]);
  at::Tensor o = at::empty({B, n, hq, D}, q.options()), lse, part;
  const bool want = truth(a[8]);
  if (want) lse = at::empty({B, n, hq}, q.options().dtype(at::kFloat));
  if (d.share) part = at::empty({d.share + problems, rows, D + 4}, q.options().dtype(at::kFloat));
  launched(k_attention(q.data_ptr(), step(q, 0), step(q, 1), step(q, 2), kp.data_ptr(), step(kp, 0), step(kp, 1), step(kp, 2),
                       vp.data_ptr(), step(vp, 0), step(vp, 1), step(vp, 2), table.data_ptr(), step(table, 0), lens.data_ptr(),
                       o.data_ptr(), want ? lse.data_ptr() : nullptr, d.share ? part.data_ptr() : nullptr, d.share ? part.numel() : 0, as_int(groups), as_int(d.share), as_int(d.least),
                       as_int(B), as_int(n), as_int(hq), as_int(hkv), as_int(D), as_int(page), as_int(width), as_int(kp.size(0)), truth(a[6]),
                       (float)scale, half_type(q.scalar_type()), w.stream),
           "dlamd_paged_attention");
  PyObject* po = THPVariable_Wrap(std::move(o));
  if (!want) return po;
  PyObject* pl = THPVariable_Wrap(std::move(lse));
  return Py_BuildValue("(NN)", po, pl);
}

// ------------------------------------------------------------------------------------------ verification
// Workgroups that share a sequence's row of `bytes` (target's and proposal's).  Up to 8192 tokens one holds it in registers
// (8 x 4000: 5.8 us, 8.0 in pieces).  128 short rows keep the card busy by themselves (256 x 32000 bf16: 14.5 us, in pieces
// 15.7), long ones are dealt out more evenly in pieces (192 x 50265 fp32: 21.0 us in 32, 21.6 in one; 512 x 50265: 38.4 and
// 42.9).  Fewer rows than compute units want more pieces (1 x 50265: 8.0 us in 48, 17 in one).
int64_t pieces_of(int64_t B, int64_t V, int64_t bytes) {
  if (V <= 8192 || (B >= 128 && bytes < 256 << 10) || B > 65535) return 1;
  return B < 32 ? std::min<int64_t>(48, (V + 511) / 512) : std::min<int64_t>(32, (V + 1535) / 1536);
}

// (draft, target, u, proposal, counts, pad, pieces or None, stream) -> (tokens, accepted)
PyObject* verify(PyObject* const* a) {
  const at::Tensor &draft = tensor(a[0]), &target = tensor(a[1]), &u = tensor(a[2]);
  const Maybe proposal = maybe(a[3]), counts = maybe(a[4]);
  need(draft.dim() == 2 && draft.scalar_type() == at::kInt, "draft is int32 [B, n]");
  const int64_t B = draft.size(0), n = draft.size(1);
  need(n <= 63, "at most 63 drafted tokens");
  const at::ScalarType dt = target.scalar_type();
  const int type = dt == at::kFloat ? 2 : half_type(dt);
  need(target.dim() == 3 && target.size(0) == B && target.size(1) == n + 1 && type >= 0 && target.size(2) > 0,
       "target is [B, n + 1, V] bf16, fp16 or fp32");
  const int64_t V = target.size(2);
  if (proposal)
    need(proposal->dim() == 3 && proposal->size(0) == B && proposal->size(1) == n && proposal->size(2) == V && proposal->scalar_type() == dt &&
             packed(*proposal.t, 2),
         "proposal is [B, n, V] of the target's type, rows contiguous");
  need(u.dim() == 2 && u.size(0) == B && u.size(1) == n + 1 && u.scalar_type() == at::kFloat && packed(u, 1), "u is fp32 [B, n + 1]");
  if (counts) need(counts->dim() == 1 && counts->size(0) == B && counts->scalar_type() == at::kInt && packed(*counts.t, 0), "counts is int32 [B]");
  need(packed(target, 2) && packed(draft, 1), "the last dimension of target and draft has to be contiguous");
  same_device(draft.device(), {&target, &u, proposal.t, counts.t});
  const ll pad = number(a[5]);
  need(pad >= -0x80000000LL && pad <= 0x7fffffffLL, "pad is an int32");
  const Where w(draft, a[7]);
  at::Tensor tokens = at::empty({B, n + 1}, draft.options()), accepted = at::empty({B}, draft.options()), sums;
  const bool with_q = proposal && n > 0;
  const int64_t pieces = a[6] == Py_None ? pieces_of(B, V, V * target.element_size() * (with_q ? 2 : 1)) : number(a[6]);
  if (pieces > 1) sums = at::empty({B, pieces, 2}, draft.options().dtype(at::kDouble));
  launched(k_verify(draft.data_ptr(), step(draft, 0), target.data_ptr(), step(target, 0), step(target, 1), with_q ? proposal.ptr() : nullptr,
                    with_q ? step(*proposal.t, 0) : 0, with_q ? step(*proposal.t, 1) : 0, u.data_ptr(), step(u, 0), counts.ptr(),
                    tokens.data_ptr(), accepted.data_ptr(), pieces > 1 ? sums.data_ptr() : nullptr, pieces > 1 ? sums.numel() : 0, as_int(pieces), as_int(B), as_int(n),
                    as_int(V), (int)pad, type, w.stream),
           "dlamd_verify_draft");
  PyObject* pt = THPVariable_Wrap(std::move(tokens));
  PyObject* pa = THPVariable_Wrap(std::move(accepted));
  return Py_BuildValue("(NN)", pt, pa);
}

// ------------------------------------------------------------------------------------------ 4-bit linear layer
struct Shape {
  int tiles, nw, kw, kz;                                     // tiles of 16 outputs per wave, waves over outputs and K, parts of K
};

// Up to 16 rows: one tile a wave and eight waves over K as long as every workgroup has a compute unit (256 tiles: 1 x 4096 x
// 4096 6.0 us, with two tiles 7.5), then two tiles that share a wave's x (16 x 6000 x 8192: 15 us, with one 21; 5 x 50265 x
// 1024: 9.7 and 11.2), with fewer waves over K where there are many (30000 x 2048: 12.0 us, with eight 12.5).
// More rows: eight tiles of products for a wave's x (four of 16 outputs, two of 16 rows) from 64 workgroups of those on
// (200 x 4096 x 4096: 31 us, with one tile of outputs 60; 64 x 2048 x 2048: 9.5 and 7.5).  Parts of K fill compute units that
// have nothing to do in the only or the last round of workgroups, for the price of sums written and read again, 4 / steps
// of the work: 128 workgroups in two parts (24 x 8192 x 28672) 41.3 us, in one 64.7; 313 in four (20 x 20000 x 8192, groups of
// 64) 40.3, in one 48.5; 188 of a shorter K in one (24 x 12000 x 4096) 18.7, in four 21.1.
Shape shape_of(int64_t M, int64_t N, int64_t K) {
  const int steps = (int)std::min<int64_t>((K + 127) / 128, 1 << 20);
  const int64_t tiles = (N + 15) / 16;
  if (M <= 16) return tiles <= 256 ? Shape{1, 1, std::min(8, steps), 1} : Shape{2, 1, std::min(tiles <= 768 ? 8 : 4, steps), 1};
  const int64_t blocks = (M + 31) / 32, wide = (tiles + 3) / 4 * blocks, groups = wide <= 64 ? tiles * blocks : wide;
  const int kw = std::min(wide <= 64 || (steps <= 8 && wide <= 256) ? 8 : 4, steps);
  auto worth = [&](int kz) {                                 // share of compute units, and of waves' steps, at work
    const int part = (steps + kz - 1) / kz, turns = (part + kw - 1) / kw;
    return (double)groups * kz / (double)((groups * kz + 255) / 256 * 256) * steps / (kz * kw * turns) - 4.0 / steps * (kz - 1);
  };
  int kz = 1;
  for (int parts = 2; parts <= std::min(4, steps) && groups <= 384; ++parts)          // beyond, rounds overlap
    if (worth(parts) > worth(kz)) kz = parts;
  return {wide <= 64 ? 1 : 4, 1, kw, kz};
}

// (x, words, scale, zero, n, k, group, bias, act, res, shape or None, stream) -> y
PyObject* int4(PyObject* const* a) {
  const at::Tensor &x = tensor(a[0]), &words = tensor(a[1]), &scale = tensor(a[2]);
  const Maybe zero = maybe(a[3]), bias = maybe(a[7]), res = maybe(a[9]);
  const int64_t N = number(a[4]), K = number(a[5]), G = number(a[6]);
  const int type = half_type(x.scalar_type());
  const int64_t dims = x.dim();
  need(dims > 0 && x.size(dims - 1) == K && type >= 0, "x is [..., K] bf16 or fp16");
  if (bias) need(bias->dim() == 1 && bias->size(0) == N && bias->scalar_type() == at::kFloat && packed(*bias.t, 0), "bias is fp32 [N]");
  if (res)
    need(res->dim() == dims && res->size(dims - 1) == N && res->sizes().slice(0, dims - 1) == x.sizes().slice(0, dims - 1) &&
             res->scalar_type() == x.scalar_type(),
         "res is [..., N] of x's type");
  need(G > 0 && K % G == 0 && words.scalar_type() == at::kInt && words.is_contiguous() && words.numel() == (N + 15) / 16 * ((K + 127) / 128) * 256 &&
           half_type(scale.scalar_type()) >= 0 && scale.is_contiguous() && scale.numel() == K / G * ((N + 15) / 16 * 16) &&
           (!zero || (zero->scalar_type() == at::kByte && zero->is_contiguous() && zero->numel() == scale.numel())),
       "words, scale and zero are not those of an [N, K] layer as pack_int4 lays it out");
  no_gradient({&x, &scale, bias.t, res.t});
  same_device(x.device(), {&words, &scale, zero.t, bias.t, res.t});
  const Where w(x, a[11]);
  at::Tensor x2 = dims == 2 ? x : x.reshape({-1, K}), r2;
  if (x2.stride(1) != 1 || step(x2, 0) % 8 != 0 || step(x2, 0) >= 1 << 24 || ((uintptr_t)x2.data_ptr() & 15))
    x2 = x2.clone(at::MemoryFormat::Contiguous);             // rows the kernel cannot load 16 bytes at a time or address
  if (res) {
    r2 = dims == 2 ? *res.t : res->reshape({-1, N});
    if (!packed(r2, 1)) r2 = r2.contiguous();
  }
  const int64_t M = x2.size(0);
  c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
  sizes[dims - 1] = N;
  at::Tensor y = at::empty(sizes, x.options()), part;
  Shape s = shape_of(M, N, K);
  if (a[10] != Py_None) {
    need(PyTuple_Check(a[10]) && PyTuple_GET_SIZE(a[10]) == 4, "shape is (tiles, waves over outputs, waves over K, parts of K)");
    s = {(int)number(PyTuple_GET_ITEM(a[10], 0)), (int)number(PyTuple_GET_ITEM(a[10], 1)), (int)number(PyTuple_GET_ITEM(a[10], 2)),
         (int)number(PyTuple_GET_ITEM(a[10], 3))};
  }
  if (s.kz > 1) part = at::empty({s.kz, M, (N + 15) / 16 * 16}, x.options().dtype(at::kFloat));
  launched(k_int4(x2.data_ptr(), step(x2, 0), words.data_ptr(), scale.data_ptr(), zero.ptr(), bias.ptr(), res ? r2.data_ptr() : nullptr,
                  res ? step(r2, 0) : 0, y.data_ptr(), as_int(M), as_int(N), as_int(K), as_int(G), (int)number(a[8]), type,
                  half_type(scale.scalar_type()), s.tiles, s.nw, s.kw, s.kz, s.kz > 1 ? part.data_ptr() : nullptr, s.kz > 1 ? part.numel() : 0, w.stream),
           "dlamd_int4_linear");
  return THPVariable_Wrap(std::move(y));
}

// ------------------------------------------------------------------------------------------ module
// No C++ exception leaves an entry: a refused argument is a ValueError, a kernel's code the framework's own error.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments are expected, %zd came", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const Failed& e) {
    PyErr_SetString(k_error ? k_error : PyExc_RuntimeError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// (address of append, attention, verify, int4, error class)
PyObject* init(PyObject* const* a) {
  auto at = [&](int i) { return (void*)(intptr_t)number(a[i]); };
  k_append = reinterpret_cast<decltype(k_append)>(at(0));
  k_attention = reinterpret_cast<decltype(k_attention)>(at(1));
  k_verify = reinterpret_cast<decltype(k_verify)>(at(2));
  k_int4 = reinterpret_cast<decltype(k_int4)>(at(3));
  Py_XINCREF(a[4]);
  k_error = a[4];
  Py_RETURN_NONE;
}
// (problems, rows, bound, D), (B, V) of fp32 rows with a proposal, (M, N, K): the rules above, for tests
PyObject* rule_deal(PyObject* const* a) {
  const Deal d = deal_out(number(a[0]), number(a[1]), number(a[2]), number(a[3]));
  return Py_BuildValue("(LL)", (ll)d.share, (ll)d.least);
}
PyObject* rule_pieces(PyObject* const* a) { return PyLong_FromLongLong(pieces_of(number(a[0]), number(a[1]), number(a[1]) * 8)); }
PyObject* rule_shape(PyObject* const* a) {
  const Shape s = shape_of(number(a[0]), number(a[1]), number(a[2]));
  return Py_BuildValue("(iiii)", s.tiles, s.nw, s.kw, s.kz);
}

#define ENTRY(name, f, n, doc) {name, (PyCFunction)(void*)entry<f, n>, METH_FASTCALL, doc}
PyMethodDef methods[] = {
    ENTRY("init", init, 5, "addresses of the kernels' C entries, the error class"),
    ENTRY("paged_append", append, 12, "ops.paged.paged_append on device tensors"),
    ENTRY("paged_attention", attention, 12, "ops.paged.paged_attention on device tensors"),
    ENTRY("verify_draft", verify, 8, "ops.draft.verify_draft on device tensors"),
    ENTRY("linear_int4", int4, 12, "ops.int4.linear_int4 on device tensors"),
    ENTRY("rule_deal", rule_deal, 4, "how attention deals its work out"),
    ENTRY("rule_pieces", rule_pieces, 2, "workgroups per row of a verification"),
    ENTRY("rule_shape", rule_shape, 3, "launch shape of a 4-bit linear layer"),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "dlamd_bind", "host side of the decode-step operators", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dlamd_bind() { return PyModule_Create(&module); }
