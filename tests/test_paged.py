"""Paged key / value cache: append with rotation and attention of new tokens, against plain 64-bit implementations."""
import math

import pytest
import torch
import torch.nn.functional as F

from distributed_llms_amd.ops import paged as P

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def cache(pages, page, hkv, D, dt, g, layout="plain"):
    """k_pages, v_pages; layout "joint": slices of one [pages, 2, page, ...] buffer, "heads": heads outside the slots."""
    if layout == "joint":
        kv = torch.randn(pages, 2, page, hkv, D, generator=g).to(dt)
        return kv[:, 0], kv[:, 1]
    if layout == "heads":
        kv = torch.randn(2, pages, hkv, page, D, generator=g).to(dt)
        return kv[0].transpose(1, 2), kv[1].transpose(1, 2)
    return tuple(torch.randn(pages, page, hkv, D, generator=g).to(dt) for _ in range(2))


def tables(need, page, g, extra=2, width=None):
    """Page table of random distinct pages for sequences of ``need`` tokens, -1 behind; (table, number of pages)."""
    counts = [-(-n // page) for n in need]
    total = sum(counts) + extra
    perm = torch.randperm(total, generator=g).to(torch.int32)
    t = torch.full((len(need), width or max([1] + counts)), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        t[b, :c] = perm[at : at + c]
        at += c
    return t, total


def gpu(*xs):
    return [None if x is None else x.cuda() for x in xs]


def on_gpu_with_strides(x):
    """A copy on the GPU with the strides of ``x`` (``.cuda()`` keeps them only for dense tensors)."""
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
    return y.copy_(x)


# ---------------------------------------------------------------------------------------------- append
def append_case(seed, need_new, kept, page, hkv, hq, D, rot, dt, interleaved, ragged, layout="plain", behind=0):
    g = torch.Generator().manual_seed(seed)
    B = len(kept)
    T = sum(need_new) + behind
    table, pages = tables([max(k, 0) + n for k, n in zip(kept, need_new)], page, g)
    kp, vp = cache(pages, page, hkv, D, dt, g, layout)
    qkv = torch.randn(T, hq + 2 * hkv, D, generator=g).to(dt)
    q, k, v = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    lens = torch.tensor(kept, dtype=torch.int32)
    starts = torch.tensor([sum(need_new[:b]) for b in range(B + 1)], dtype=torch.int32) if ragged else None
    cos, sin = P.rope_tables(table.shape[1] * page, rot) if rot else (None, None)
    return dict(k=k, v=v, k_pages=kp, v_pages=vp, table=table, lens=lens, q=q if hq else None, cos=cos, sin=sin, starts=starts,
                interleaved=interleaved)


def close_half_step(got, ref, dt):
    """One rounding (half a step of ``dt``) of fp32 maths whose own error is a few fp32 steps of the operands (|x| < 8)."""
    err = (got.double() - ref.double()).abs()
    tol = torch.finfo(dt).eps / 2 * ref.double().abs() + 32 * 2.0 ** -24
    assert bool((err <= tol).all()), float((err - tol).max())


def rotate64(x, pos, rot, interleaved):
    """Rotation as complex numbers, angles from the position in 64 bits."""
    x = x.double()
    if rot == 0:
        return x
    w = torch.polar(torch.ones(rot // 2, dtype=torch.float64), pos * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot))
    r = x[..., :rot]
    if interleaved:
        z = torch.view_as_complex(r.reshape(*r.shape[:-1], rot // 2, 2).contiguous()) * w
        y = torch.view_as_real(z).reshape(r.shape)
    else:
        z = torch.complex(r[..., : rot // 2].contiguous(), r[..., rot // 2 :].contiguous()) * w
        y = torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., rot:]), -1)


def check_append(c, got_k, got_v, got_q, rot):
    """Expected cache and queries token by token from the definition."""
    B, (pages, page) = len(c["lens"]), c["k_pages"].shape[:2]
    T = c["k"].shape[0]
    dt = c["k"].dtype
    kp, vp = c["k_pages"].double().clone(), c["v_pages"].double().clone()
    qo = torch.zeros(c["q"].shape, dtype=torch.float64) if c["q"] is not None else None
    starts = c["starts"].tolist() if c["starts"] is not None else [T // B * b for b in range(B + 1)]
    written = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(B):
        for t in range(starts[b], min(starts[b + 1], T)):
            pos = int(c["lens"][b]) + t - starts[b]
            if int(c["lens"][b]) < 0 or pos >= c["table"].shape[1] * page:
                continue
            if qo is not None:
                qo[t] = rotate64(c["q"][t], pos, rot, c["interleaved"])
            pid = int(c["table"][b, pos // page])
            if 0 <= pid < pages:
                kp[pid, pos % page] = rotate64(c["k"][t], pos, rot, c["interleaved"])
                vp[pid, pos % page] = c["v"][t].double()
                written[pid, pos % page] = True
    assert torch.equal(got_v.double(), vp)
    assert torch.equal(got_k.double()[~written], kp[~written])          # what was there stays, bit for bit
    # angles of far positions: the table holds them to half a fp32 step, so a rotated value is off by |x| 2^-24 more
    close_half_step(got_k, kp, dt)
    if qo is not None:
        close_half_step(got_q, qo, dt)


APPEND = [
    # need_new, kept, page, hkv, hq, D, rot, dtype, interleaved, ragged, layout, behind
    ([1], [0], 16, 1, 0, 64, 0, "bf16", False, False, "plain", 0),
    ([1] * 5, [0, 15, 16, 31, 200], 16, 16, 0, 64, 0, "bf16", False, False, "plain", 0),
    ([5] * 3, [0, 13, 63], 64, 8, 32, 128, 128, "fp16", False, False, "joint", 0),
    ([4] * 4, [-1, 3, -7, 0], 16, 2, 4, 64, 32, "bf16", True, False, "plain", 0),
    ([7, 0, 33, 1, 0], [0, 5, 40, 100, 3], 48, 2, 6, 64, 16, "bf16", False, True, "heads", 9),
    ([0, 0, 3], [0, 0, 0], 16, 1, 1, 128, 64, "fp16", True, True, "plain", 0),
    ([130, 1, 77], [9000, 0, 31], 128, 3, 3, 128, 128, "bf16", True, True, "joint", 64),
    ([2] * 70, [i * 3 for i in range(70)], 8, 1, 2, 72, 48, "bf16", False, True, "plain", 3),
    ([3] * 200, [(i * 37) % 90 for i in range(200)], 5, 2, 2, 64, 64, "fp16", False, True, "plain", 0),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_oracle(case):
    n, kept, page, hkv, hq, D, rot, dt, il, ragged, layout, behind = APPEND[case]
    c = append_case(case, n, kept, page, hkv, hq, D, rot, DTYPES[dt], il, ragged, layout, behind)
    kp, vp = c["k_pages"].clone(), c["v_pages"].clone()
    qo = P.paged_append(**{**c, "k_pages": kp, "v_pages": vp})
    check_append(c, kp, vp, qo, rot)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_kernel(case):
    n, kept, page, hkv, hq, D, rot, dt, il, ragged, layout, behind = APPEND[case]
    c = append_case(case, n, kept, page, hkv, hq, D, rot, DTYPES[dt], il, ragged, layout, behind)
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    full = torch.empty((c["k"].shape[0], hq + 2 * hkv, D), dtype=DTYPES[dt], device="cuda")       # slices of one projection
    full[:, hq : hq + hkv], full[:, hq + hkv :] = c["k"].cuda(), c["v"].cuda()
    if hq:
        full[:, :hq] = c["q"].cuda()
        d["q"] = full[:, :hq]
    d["k"], d["v"] = full[:, hq : hq + hkv], full[:, hq + hkv :]
    d["k_pages"], d["v_pages"] = on_gpu_with_strides(c["k_pages"]), on_gpu_with_strides(c["v_pages"])
    before = full.clone()
    qo = P.paged_append(**d)
    assert torch.equal(full, before)
    check_append(c, d["k_pages"].cpu(), d["v_pages"].cpu(), None if qo is None else qo.cpu(), rot)


def bad_table_case():
    c = append_case(3, [4] * 4, [0, 14, 30, 2], 16, 2, 2, 64, 64, torch.bfloat16, False, False)
    c["table"] = torch.tensor([[-1, 0, 0], [0, 1 << 30, 0], [1, 2, -(1 << 31)], [c["k_pages"].shape[0], 0, 0]], dtype=torch.int32)
    c["cos"], c["sin"] = P.rope_tables(48, 64)
    return c


def test_append_to_missing_pages_writes_nothing():
    c = bad_table_case()
    kp, vp = c["k_pages"].clone(), c["v_pages"].clone()
    qo = P.paged_append(**{**c, "k_pages": kp, "v_pages": vp})
    check_append(c, kp, vp, qo, 64)


@pytest.mark.gpu
def test_append_kernel_to_missing_pages_writes_nothing():
    c = bad_table_case()
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    qo = P.paged_append(**d)
    check_append(c, d["k_pages"].cpu(), d["v_pages"].cpu(), qo.cpu(), 64)


def test_rope_tables_are_exact_at_far_positions():
    cos, sin = P.rope_tables(200001, 16)
    ang = 200000 * 10000.0 ** (-2.0 / 16)
    assert abs(float(cos[200000, 1]) - math.cos(ang)) <= 2.0 ** -24 and abs(float(sin[200000, 1]) - math.sin(ang)) <= 2.0 ** -24


# ---------------------------------------------------------------------------------------------- attention
def att_case(seed, kept, n, page, hq, hkv, D, dt, causal, layout="plain", qscale=1.5):
    g = torch.Generator().manual_seed(seed)
    need = [max(k, 0) + (n if causal and k >= 0 else 0) for k in kept]
    table, pages = tables(need, page, g)
    kp, vp = cache(pages, page, hkv, D, dt, g, layout)
    # slots nobody has written hold NaN and infinities
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, m in enumerate(need):
        for p in range(m):
            used[int(table[b, p // page]), p % page] = True
    kp[~used] = float("nan")
    vp[~used] = float("inf")
    q = (torch.randn(len(kept), n, hq, D, generator=g) * qscale).to(dt)
    return dict(q=q, k_pages=kp, v_pages=vp, table=table, lens=torch.tensor(kept, dtype=torch.int32), causal=causal)


def att_tolerance(c, ref):
    """Half a step of the output's type, plus the fp32 maths: scores |s| < 64 carry 2^-24 |s| (D + 2) in the worst case of
    their sum, which the exponential turns into that relative error; the weights are kept to 2^-16."""
    vmax = c["v_pages"].double().nan_to_num(0, 0, 0).abs().max()
    return torch.finfo(c["q"].dtype).eps / 2 * ref.abs() + float(vmax) * 2.0 ** -13


def check_attention(c, o, lse):
    ref, ref_lse = P.paged_attention_reference(**c, dtype=torch.float64)
    assert o.dtype == c["q"].dtype and o.shape == c["q"].shape and lse.dtype == torch.float32
    err = (o.double() - ref).abs()
    assert bool((err <= att_tolerance(c, ref)).all()), float(err.max())
    empty = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse.double()), empty) and bool((lse[empty] < 0).all()) and bool((o[empty] == 0).all())
    assert bool(((lse.double() - ref_lse).abs()[~empty] <= 2.0 ** -24 * 130 * 64).all())


ATT = [
    # kept, n, page, hq, hkv, D, dtype, causal, layout
    ([0], 1, 16, 1, 1, 64, "bf16", True, "plain"),
    ([0, 1, 30, 31, 32, 127], 1, 16, 4, 4, 64, "bf16", True, "plain"),
    ([0, -1, 5, 64], 1, 32, 2, 2, 64, "bf16", False, "joint"),
    ([577] * 3, 1, 32, 16, 16, 64, "bf16", False, "plain"),
    ([100, 0, 47, 48, 1000], 5, 48, 32, 4, 128, "fp16", True, "joint"),
    ([3, 2500], 3, 16, 6, 2, 128, "bf16", True, "heads"),
    ([4999], 1, 64, 32, 8, 128, "bf16", True, "plain"),
    ([20011, 7], 2, 80, 4, 1, 64, "fp16", True, "plain"),
    ([17, 300], 16, 16, 24, 2, 128, "bf16", True, "plain"),
    ([33, 0, 600], 9, 256, 7, 1, 64, "fp16", False, "heads"),
    ([9] * 70, 2, 16, 4, 2, 64, "bf16", True, "plain"),
    ([700], 40, 32, 5, 1, 64, "bf16", True, "plain"),
    ([300, 2], 10, 16, 8, 1, 128, "bf16", True, "plain"),
    ([(i * 61) % 400 - 1 for i in range(130)], 1, 16, 3, 1, 64, "fp16", True, "joint"),
]


@pytest.mark.parametrize("case", [0, 2, 4, 9])
def test_attention_oracle_against_dense_attention(case):
    kept, n, page, hq, hkv, D, dt, causal, layout = ATT[case]
    c = att_case(case, kept, n, page, hq, hkv, D, DTYPES[dt], causal, layout)
    o, lse = P.paged_attention(**c, return_lse=True)
    check_attention(c, o, lse)
    for b, m in enumerate(kept):
        for i in range(n):
            seen = max(m, 0) + (i + 1 if causal and m >= 0 else 0)
            if seen == 0:
                continue
            pos = torch.arange(seen)
            pid = c["table"][b].long()[pos // page]
            k, v = (x[pid, pos % page].double().repeat_interleave(hq // hkv, 1).transpose(0, 1) for x in (c["k_pages"], c["v_pages"]))
            ref = F.scaled_dot_product_attention(c["q"][b, i].double()[:, None], k, v)[:, 0]
            assert bool(((o[b, i].double() - ref).abs() <= att_tolerance(c, ref)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(ATT)))
def test_attention_kernel(case):
    kept, n, page, hq, hkv, D, dt, causal, layout = ATT[case]
    c = att_case(case, kept, n, page, hq, hkv, D, DTYPES[dt], causal, layout)
    d = {x: on_gpu_with_strides(y) if torch.is_tensor(y) else y for x, y in c.items()}
    o, lse = P.paged_attention(**d, return_lse=True)
    check_attention(c, o.cpu(), lse.cpu())
    assert torch.equal(P.paged_attention(**d), o)                     # without the log-sum-exp, and again: the same bits


def missing_pages_case():
    c = att_case(11, [100, 60, 33], 2, 16, 8, 2, 64, torch.bfloat16, True)
    c["table"][0, 2] = -1                       # a hole
    c["table"][1] = torch.tensor(c["k_pages"].shape[0], dtype=torch.int32)      # no page at all
    c["table"][2, 0] = 1 << 30
    return c


def test_attention_oracle_skips_missing_pages():
    c = missing_pages_case()
    o, lse = P.paged_attention(**c, return_lse=True)
    check_attention(c, o, lse)
    assert bool((o[1] == 0).all()) and not bool((o[0] == 0).all())


@pytest.mark.gpu
def test_attention_kernel_skips_missing_pages():
    c = missing_pages_case()
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o, lse = P.paged_attention(**d, return_lse=True)
    check_attention(c, o.cpu(), lse.cpu())


def peaked_case():
    """Scores from -600 to 600: one key takes everything, and it lies near the end, in the middle or in front."""
    c = att_case(5, [400, 390, 380], 1, 16, 4, 2, 64, torch.bfloat16, True, qscale=1.0)
    for b, at in enumerate((399, 200, 0)):
        pid = int(c["table"][b, at // 16])
        c["k_pages"][pid, at % 16] = (c["q"][b, 0].view(2, 2, 64)[:, 0].float() * 8).to(torch.bfloat16)
    c["q"] = (c["q"].float() * 8).to(torch.bfloat16)
    return c


@pytest.mark.gpu
def test_attention_kernel_with_peaked_scores():
    c = peaked_case()
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o, lse = (x.cpu() for x in P.paged_attention(**d, return_lse=True))
    ref, ref_lse = P.paged_attention_reference(**c, dtype=torch.float64)
    assert torch.isfinite(o).all()
    # scores up to 700 carry 2^-24 * 700 * 66 < 2^-8.5 absolute error in the worst case, as relative error of the weights
    vmax = float(c["v_pages"].double().nan_to_num(0, 0, 0).abs().max())
    assert bool(((o.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + vmax * 2.0 ** -8).all())
    assert bool(((lse.double() - ref_lse).abs() <= 2.0 ** -8).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.1, 0.02, 1.5])
def test_attention_kernel_with_other_scales(scale):
    c = att_case(8, [90, 300], 2, 16, 4, 2, 64, torch.bfloat16, True, qscale=0.3)
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o, lse = P.paged_attention(**d, scale=scale, return_lse=True)
    ref, ref_lse = P.paged_attention_reference(**c, scale=scale, dtype=torch.float64)
    assert bool(((o.cpu().double() - ref).abs() <= att_tolerance(c, ref)).all())
    assert bool(((lse.cpu().double() - ref_lse).abs() <= 2.0 ** -24 * 130 * 64).all())


@pytest.mark.gpu
def test_attention_kernel_with_infinite_and_nan_keys_in_sight():
    """A visible key whose score is -inf weighs nothing; a NaN in a visible value reaches its own row only."""
    c = att_case(6, [50, 50], 1, 16, 2, 2, 64, torch.bfloat16, True)
    c["q"] = c["q"].abs() + 0.1
    c["q"] = c["q"].to(torch.bfloat16)
    c["k_pages"][int(c["table"][0, 1]), 3] = float("-inf")
    c["v_pages"][int(c["table"][1, 1]), 3, 0, 5] = float("nan")
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o = P.paged_attention(**d).cpu()
    ref, _ = P.paged_attention_reference(**c, dtype=torch.float64)
    assert bool(((o[0].double() - ref[0]).abs() <= att_tolerance(c, ref[0])).all())
    nan = torch.isnan(o)
    assert bool(nan[1, 0, 0, 5]) and int(nan.sum()) == 1


def odd_values_case(dt):
    """NaN and infinities in the values of the newest tokens: rows of earlier tokens do not see them."""
    c = att_case(13, [63, 90, 400], 6, 16, 16, 2, 128, dt, True)
    for b, (i, d, x) in enumerate(((1, 0, float("nan")), (5, 127, float("inf")), (3, 64, float("-inf")))):
        pos = int(c["lens"][b]) + i
        c["v_pages"][int(c["table"][b, pos // 16]), pos % 16, :, d] = x
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_attention_kernel_keeps_odd_values_from_rows_that_do_not_see_them(dt):
    c = odd_values_case(DTYPES[dt])
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o = P.paged_attention(**d).cpu()
    ref, _ = P.paged_attention_reference(**c, dtype=torch.float64)
    for b, (i, dim) in enumerate(((1, 0), (5, 127), (3, 64))):
        assert torch.isfinite(o[b, :i]).all() and not torch.isfinite(o[b, i:, :, dim]).any()
        assert torch.isfinite(o[b, i:].double()).sum() == torch.isfinite(ref[b, i:]).sum()
    ok = torch.isfinite(ref)
    assert torch.equal(torch.isnan(o), torch.isnan(ref)) and torch.equal(o[~ok].isinf(), ref[~ok].isinf())
    vmax = float(c["v_pages"].double().nan_to_num(0, 0, 0).abs().max())
    assert bool(((o.double() - ref).abs()[ok] <= torch.finfo(DTYPES[dt]).eps / 2 * ref.abs()[ok] + vmax * 2.0 ** -13).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", [2, 4, 6, 7, 8, 10, 11, 12, 13])
@pytest.mark.parametrize("share,least", [(0, 0), (1, 1), (2, 1), (7, 3), (64, 1), (700, 1), (256, 100000)])
def test_attention_kernel_shares(case, share, least, monkeypatch):
    """Any way of dealing the work out gives the result: one workgroup for all of it, borders inside sequences, heads and
    groups of rows, more workgroups than tiles."""
    kept, n, page, hq, hkv, D, dt, causal, layout = ATT[case]
    c = att_case(case, kept, n, page, hq, hkv, D, DTYPES[dt], causal, layout)
    d = {x: on_gpu_with_strides(y) if torch.is_tensor(y) else y for x, y in c.items()}
    monkeypatch.setattr(P, "_DEAL", (share, least))
    o, lse = P.paged_attention(**d, return_lse=True)
    check_attention(c, o.cpu(), lse.cpu())


@pytest.mark.gpu
def test_attention_kernel_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements (4.3 GB each of K and V): the sequence's pages lie at both ends."""
    page, hkv, D = 256, 8, 128
    pages = (1 << 31) // (page * hkv * D) + 8
    kp = torch.zeros((pages, page, hkv, D), dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    g = torch.Generator().manual_seed(9)
    small_k, small_v = (torch.randn(3, page, hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    where = [pages - 1, 0, pages - 3]
    for j, pid in enumerate(where):
        kp[pid], vp[pid] = small_k[j].cuda(), small_v[j].cuda()
    new_k, new_v = (torch.randn(1, hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([where], dtype=torch.int32)
    lens = torch.tensor([700], dtype=torch.int32)
    q = torch.randn(1, 1, 16, D, generator=g).to(torch.bfloat16)
    P.paged_append(new_k.cuda(), new_v.cuda(), kp, vp, table.cuda(), lens.cuda())
    o = P.paged_attention(q.cuda(), kp, vp, table.cuda(), lens.cuda()).cpu()
    small_k[2, 700 - 512], small_v[2, 700 - 512] = new_k[0], new_v[0]
    c = dict(q=q, k_pages=small_k, v_pages=small_v, table=torch.tensor([[0, 1, 2]], dtype=torch.int32), lens=lens, causal=True)
    ref, _ = P.paged_attention_reference(**c, dtype=torch.float64)
    assert bool(((o.double() - ref).abs() <= att_tolerance(c, ref)).all())
    del kp, vp
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_nothing_to_do():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    assert P.paged_attention(z(0, 1, 2, 64), z(1, 16, 2, 64), z(1, 16, 2, 64), i(0, 1), i(0)).shape == (0, 1, 2, 64)
    assert P.paged_attention(z(2, 0, 2, 64), z(1, 16, 2, 64), z(1, 16, 2, 64), i(2, 1), i(2)).numel() == 0
    o, lse = P.paged_attention(z(2, 1, 2, 64) + 1, z(1, 16, 2, 64), z(1, 16, 2, 64), i(2, 0), i(2), return_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    o = P.paged_attention(z(2, 1, 2, 64) + 1, z(0, 16, 2, 64), z(0, 16, 2, 64), i(2, 3), i(2) + 9)
    assert bool((o == 0).all())
    kp = z(1, 16, 2, 64)
    assert P.paged_append(z(0, 2, 64), z(0, 2, 64), kp, kp.clone(), i(3, 1), i(3)) is None
    q = P.paged_append(z(3, 2, 64) + 1, z(3, 2, 64), kp, kp.clone(), i(3, 0), i(3), q=z(3, 2, 64) + 1)
    assert bool((q == 0).all()) and bool((kp == 0).all())


# ---------------------------------------------------------------------------------------------- refusals
def _append_args():
    c = append_case(1, [2] * 2, [0, 3], 16, 2, 4, 64, 32, torch.bfloat16, False, False)
    return c


APPEND_REFUSED = {
    "types differ": lambda c: c.update(k=c["k"].half()),
    "cache types differ": lambda c: c.update(v_pages=c["v_pages"].half()),
    "fp32 cache": lambda c: c.update(k_pages=c["k_pages"].float(), v_pages=c["v_pages"].float()),
    "heads differ": lambda c: c.update(k=c["k"][:, :1], v=c["v"][:, :1]),
    "not one token count": lambda c: c.update(v=c["v"][:2]),
    "uneven without starts": lambda c: c.update(k=c["k"][:3], v=c["v"][:3], q=None),
    "short rotation tables": lambda c: c.update(cos=c["cos"][:5], sin=c["sin"][:5]),
    "cos without sin": lambda c: c.update(sin=None),
    "odd rotation": lambda c: c.update(cos=c["cos"][:, :5], sin=c["sin"][:, :5]),
    "rotation beyond D": lambda c: c.update(cos=torch.zeros(64, 40), sin=torch.zeros(64, 40)),
    "64-bit lens": lambda c: c.update(lens=c["lens"].long()),
    "64-bit table": lambda c: c.update(table=c["table"].long()),
    "lens of another batch": lambda c: c.update(lens=c["lens"][:1]),
    "starts of another batch": lambda c: c.update(starts=torch.zeros(2, dtype=torch.int32)),
    "last dimension strided": lambda c: c.update(k=c["k"].transpose(0, 2).contiguous().transpose(0, 2)),
    "q of another type": lambda c: c.update(q=c["q"].half()),
    "q of another length": lambda c: c.update(q=c["q"][:2]),
}


@pytest.mark.parametrize("why", sorted(APPEND_REFUSED))
def test_append_refuses(why):
    c = _append_args()
    APPEND_REFUSED[why](c)
    with pytest.raises(ValueError):
        P.paged_append(**c)


ATT_REFUSED = {
    "types differ": lambda c: c.update(q=c["q"].half()),
    "heads no multiple": lambda c: c.update(q=c["q"][:, :, :3]),
    "page 8": lambda c: c.update(k_pages=c["k_pages"][:, :8], v_pages=c["v_pages"][:, :8]),
    "D 32": lambda c: c.update(q=c["q"][..., :32], k_pages=c["k_pages"][..., :32], v_pages=c["v_pages"][..., :32]),
    "D differs": lambda c: c.update(q=c["q"][..., :32]),
    "table of another batch": lambda c: c.update(table=c["table"][:1], lens=c["lens"][:1]),
    "64-bit lens": lambda c: c.update(lens=c["lens"].long()),
    "one query, no n": lambda c: c.update(q=c["q"][:, 0]),
    "K and V differ": lambda c: c.update(v_pages=c["v_pages"][:1]),
}


@pytest.mark.parametrize("why", sorted(ATT_REFUSED))
def test_attention_refuses(why):
    c = att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True)
    ATT_REFUSED[why](c)
    with pytest.raises(ValueError):
        P.paged_attention(**c)


@pytest.mark.gpu
def test_kernels_refuse_what_they_cannot_load():
    """Misaligned rows (16 bytes at a time) and a misplaced tensor are refused on the host, nothing is launched."""
    from distributed_llms_amd.ops._loader import KernelLibraryError

    c = att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True)
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    q = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 1, 4, 64)
    with pytest.raises(KernelLibraryError):
        P.paged_attention(**{**d, "q": q})
    with pytest.raises(ValueError):
        P.paged_attention(**{**d, "lens": c["lens"]})
    odd = torch.zeros(2, 2, 65, dtype=torch.bfloat16, device="cuda")[..., :64]
    with pytest.raises(KernelLibraryError):
        P.paged_append(odd, odd, d["k_pages"], d["v_pages"], d["table"], d["lens"])
    with pytest.raises(ValueError):
        P.paged_append(odd.cpu(), odd.cpu(), d["k_pages"], d["v_pages"], d["table"], d["lens"])


BINDING = ["checks", pytest.param("cuda", marks=pytest.mark.gpu)]     # "checks": the device path's host checks, on CPU tensors


def refused_by_the_binding(dev, c, call):
    """The host side for device tensors refuses before it launches, so its checks can be seen without a GPU too."""
    from distributed_llms_amd.ops import _loader

    if dev == "checks" and not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    with pytest.raises(ValueError):
        call(_loader.bind(), {n: x.cuda() if dev == "cuda" and torch.is_tensor(x) else x for n, x in c.items()})


MORE_APPEND_REFUSED = {
    **APPEND_REFUSED,
    "keys that require a gradient": lambda c: c.update(k=c["k"].clone().requires_grad_()),
    "queries that require a gradient": lambda c: c.update(q=c["q"].clone().requires_grad_()),
    "a cache without heads": lambda c: c.update(k=c["k"][:, :0], v=c["v"][:, :0], k_pages=c["k_pages"][:, :, :0], v_pages=c["v_pages"][:, :, :0]),
    "queries without heads": lambda c: c.update(q=c["q"][:, :0]),
}
MORE_ATT_REFUSED = {
    **ATT_REFUSED,
    "queries that require a gradient": lambda c: c.update(q=c["q"].clone().requires_grad_()),
    "a cache that requires a gradient": lambda c: c.update(v_pages=c["v_pages"].clone().requires_grad_()),
    "an infinite scale": lambda c: c.update(scale=math.inf),
    "no scale at all": lambda c: c.update(scale=math.nan),
    "a scale beyond fp32": lambda c: c.update(scale=1e39),
}


@pytest.mark.parametrize("dev", BINDING)
@pytest.mark.parametrize("why", sorted(MORE_APPEND_REFUSED))
def test_append_refuses_on_the_device_path(why, dev):
    c = {"q": None, "cos": None, "sin": None, "starts": None, "interleaved": False, **_append_args()}
    MORE_APPEND_REFUSED[why](c)
    with pytest.raises(ValueError):
        P.paged_append(**c)
    refused_by_the_binding(dev, c, lambda bind, d: bind.paged_append(
        *(d[x] for x in ("k", "v", "k_pages", "v_pages", "table", "lens", "q", "cos", "sin", "starts", "interleaved")), 0))


@pytest.mark.parametrize("dev", BINDING)
@pytest.mark.parametrize("why", sorted(MORE_ATT_REFUSED))
def test_attention_refuses_on_the_device_path(why, dev):
    c = {"scale": None, "causal": True, **att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True)}
    MORE_ATT_REFUSED[why](c)
    with pytest.raises(ValueError):
        P.paged_attention(**c)
    refused_by_the_binding(dev, c, lambda bind, d: bind.paged_attention(
        *(d[x] for x in ("q", "k_pages", "v_pages", "table", "lens", "scale", "causal")), None, False, None, 0, 0))


@pytest.mark.parametrize("dev", BINDING)
def test_the_device_path_wants_tensors_and_numbers(dev):
    c = {"scale": None, "causal": True, **att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True)}
    for bad in (dict(scale="large"), dict(q=3), dict(lens=None)):
        refused_by_the_binding(dev, {**c, **bad}, lambda bind, d: bind.paged_attention(
            *(d[x] for x in ("q", "k_pages", "v_pages", "table", "lens", "scale", "causal")), None, False, None, 0, 0))


def test_no_gradient_is_asked_for_under_no_grad():
    c = att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True)
    want = P.paged_attention(**c)
    with torch.no_grad():
        assert torch.equal(P.paged_attention(**{**c, "q": c["q"].clone().requires_grad_()}), want)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_row_with_nothing_but_scores_of_minus_infinity(dev):
    """As if it saw nothing; the row of the next token sees one key more, and only that."""
    c = att_case(6, [1, 40], 2, 16, 2, 2, 64, torch.bfloat16, True)
    c["q"] = (c["q"].abs() + 0.1).to(torch.bfloat16)
    for pos in (0, 1):
        c["k_pages"][int(c["table"][0, 0]), pos] = float("-inf")
    first = c["lens"].clone()
    first[0] = 0
    for lens in (c["lens"], first):
        c["lens"] = lens
        d = {x: y.to(dev) if torch.is_tensor(y) else y for x, y in c.items()}
        o, lse = P.paged_attention(**d, return_lse=True)
        ref, ref_lse = P.paged_attention_reference(**c, dtype=torch.float64)
        rows = 2 - int(lens[0])                                      # those that see positions 0 and 1 at most
        assert bool((o[0, :rows].cpu() == 0).all()) and bool(torch.isneginf(lse[0, :rows].cpu()).all())
        assert bool(((o.cpu().double() - ref).abs() <= att_tolerance(c, ref)).all())
    c["k_pages"][int(c["table"][0, 0]), 1] = 0.5
    d = {x: y.to(dev) if torch.is_tensor(y) else y for x, y in c.items()}
    o = P.paged_attention(**d).cpu()
    assert bool((o[0, 0] == 0).all()) and torch.equal(o[0, 1], c["v_pages"][int(c["table"][0, 0]), 1])


def test_c_entries_refuse_more_than_a_launch_holds():
    """Sizes whose grids would have 2^32 threads, and workspaces that are too small; refused before anything is read."""
    import ctypes

    from distributed_llms_amd.ops import _loader

    if not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    lib = _loader.lib()
    i, ll, p = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p
    z, at = p(0), p(1 << 20)

    def append(T):
        return lib.dlamd_paged_append(at, ll(64), ll(64), at, ll(64), ll(64), z, ll(0), ll(0), z, at, ll(1024), ll(64), ll(64), at, ll(1024),
                                      ll(64), ll(64), at, ll(1), at, z, z, z, i(1), i(T), i(0), i(1), i(64), i(0), i(16), i(1), i(0), i(0),
                                      i(0), z)

    def attention(B, n, share, floats):
        return lib.dlamd_paged_attention(at, ll(64), ll(64), ll(64), at, ll(1024), ll(64), ll(64), at, ll(1024), ll(64), ll(64), at, ll(1),
                                         at, at, z, at, ll(floats), i(1), i(share), i(1), i(B), i(n), i(1), i(1), i(64), i(16), i(1), i(1), i(0),
                                         ctypes.c_float(1), i(0), z)

    assert append(1 << 24) == -8
    assert attention(1 << 24, 1, 0, 0) == -10 and attention(1 << 12, 1 << 12, 8, 1 << 60) == -9
    assert attention(4, 1, 8, 100) == -12


@pytest.mark.gpu
@pytest.mark.parametrize("share,least", [(None, 0), (0, 0), (1, 1), (37, 1), (256, 1), (256, 9)])
@pytest.mark.parametrize("n,hq,hkv,D,dt", [(5, 16, 2, 128, "fp16"), (5, 16, 2, 64, "bf16"), (3, 30, 2, 128, "bf16"), (11, 8, 2, 64, "fp16")])
def test_attention_kernel_with_three_tiles_of_rows(n, hq, hkv, D, dt, share, least, monkeypatch):
    """33 to 48 rows stay together where the cache may be long: a wide table that is mostly empty.  A tight bound splits them,
    and the result is right either way."""
    monkeypatch.setattr(P, "_DEAL", (share, least))
    c = att_case(31, [400, 0, -1, 47, 1, 300, 129, 128], n, 16, hq, hkv, D, DTYPES[dt], True)
    c["table"] = torch.cat((c["table"], torch.full((8, 1024), -1, dtype=torch.int32)), 1)
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    for bound in (None, 500):
        o, lse = P.paged_attention(**d, return_lse=True, max_len=bound)
        check_attention(c, o.cpu(), lse.cpu())


# ---------------------------------------------------------------------------------------------- weights over their whole range
def far_case(size, sign, dt, seed=0):
    """Scores around sign * size: keys are multiples of the signs of q, one of them a seventh or more above all others."""
    g = torch.Generator().manual_seed(seed)
    B, hkv, G, D, page, kept = 24, 2, 3, 64, 16, 300
    table, pages = tables([kept] * B, page, g)
    vp = torch.randn(pages, page, hkv, D, generator=g).to(dt)
    signs = torch.randint(0, 2, (B, hkv, D), generator=g) * 2.0 - 1.0
    level = (size * 8 / D) ** 0.5                                # scale is 1 / 8
    q = signs[:, :, None] * level * (1 + torch.randint(0, 16, (B, hkv, G, 1), generator=g) / 16)
    kp = torch.zeros(pages, page, hkv, D)
    for b in range(B):
        steps = 1 + torch.randint(16, 48, (kept,), generator=g) / 64
        steps[int(torch.randint(0, kept, (1,), generator=g))] = 1 + 63 / 64 if sign > 0 else 1.0
        for p in range(kept):
            kp[int(table[b, p // page]), p % page] = sign * signs[b] * level * steps[p]
    return dict(q=q.reshape(B, 1, hkv * G, D).to(dt), k_pages=kp.to(dt), v_pages=vp, table=table,
                lens=torch.full((B,), kept, dtype=torch.int32), causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dt,size", [("bf16", 2.0 ** e) for e in (12, 24, 28, 32, 36, 60, 100)] + [("fp16", 2.0 ** e) for e in (12, 24, 28, 31)])
@pytest.mark.parametrize("share", [0, 64])
def test_attention_kernel_with_far_scores(dt, size, sign, share, monkeypatch):
    """The largest score is hundreds above the next, so one key is the result: its value (a product with its weight and a
    division by it: two fp32 roundings).  The log-sum-exp is that score: D + 4 roundings of 2^-24."""
    monkeypatch.setattr(P, "_DEAL", (share, 1))
    c = far_case(size, sign, DTYPES[dt])
    ref, ref_lse = P.paged_attention_reference(**c, dtype=torch.float64)
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o, lse = (x.cpu() for x in P.paged_attention(**d, return_lse=True))
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    assert bool(((o.double() - ref).abs() <= 2.0 ** -20 * ref.abs()).all())
    assert bool(((lse.double() - ref_lse).abs() <= 2.0 ** -24 * 68 * ref_lse.abs()).all())


def sink_case(gap, kept, dt, D, at):
    """One key `gap` nats above all others, with a value of zero: the result is what the small weights add up to.  q is all
    ones and the sink's key all gap / D, so its score is exact; the others' scores lie within a few tenths of zero, their
    values between 0.5 and 1.5."""
    g = torch.Generator().manual_seed(gap * 1000 + kept)
    page, hkv, G = 16, 2, 2
    table, pages = tables([kept] * 2, page, g)
    kp = (torch.randn(pages, page, hkv, D, generator=g) * 0.02).to(dt)
    vp = (torch.rand(pages, page, hkv, D, generator=g) + 0.5).to(dt)
    for b in range(2):
        pos = (at, kept - 1 - at)[b]
        kp[int(table[b, pos // page]), pos % page] = gap / D
        vp[int(table[b, pos // page]), pos % page] = 0.0
    return dict(q=torch.ones(2, 1, hkv * G, D, dtype=dt), k_pages=kp, v_pages=vp, table=table,
                lens=torch.full((2,), kept, dtype=torch.int32), causal=False, scale=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("gap,kept,D,at", [(10, 200, 64, 3), (12, 4096, 128, 1000), (14, 32, 64, 7), (14, 4096, 64, 2048), (16, 32, 128, 0),
                                           (16, 20000, 64, 17), (20, 4096, 64, 4095), (24, 20000, 128, 9999)])
@pytest.mark.parametrize("share", [0, 64, None])
def test_attention_kernel_keeps_small_weights(gap, kept, D, at, dt, share, monkeypatch):
    """Tolerance: half a step of the result, and relative to sum p |v| (the result itself: values are positive): the sink's score
    and a key's are each off by (D + 2) 2^-24 of the sum of |q k| (gap, and less than 2.5), the split of a weight into
    two numbers of 16 bits by 2^-16, the fp32 sums and the exponential by 2^-18."""
    if share is not None:
        monkeypatch.setattr(P, "_DEAL", (share, 1))
    c = sink_case(gap, kept, DTYPES[dt], D, at)
    ref, ref_lse = P.paged_attention_reference(**c, dtype=torch.float64)
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o, lse = (x.cpu().double() for x in P.paged_attention(**d, return_lse=True))
    weight = 2.0 ** -24 * (D + 2) * (gap + 2.5) + 2.0 ** -16 + 2.0 ** -18
    step = torch.finfo(DTYPES[dt]).eps / 2 * ref.abs() + (2.0 ** -25 if dt == "fp16" else 0.0)       # fp16's last step is 2^-24
    err, tol = (o - ref).abs(), step + weight * ref.abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    assert bool(((lse - ref_lse).abs() <= 2.0 ** -24 * (D + 8) * (gap + 2.5)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("share", [0, 64])
def test_attention_kernel_with_an_odd_value_and_large_scores(dt, share, monkeypatch):
    """NaN in one dimension of one visible value leaves the others alone, also where scores are large: a rounding of theirs is
    then no small part of a weight, and weights and their sum have to come from the same scores.  One key stands out, so the
    other dimensions are its value's."""
    monkeypatch.setattr(P, "_DEAL", (share, 1))
    dtype, g = DTYPES[dt], torch.Generator().manual_seed(3)
    c = att_case(21, [90, 200, 33, 64], 1, 16, 8, 2, 64, dtype, False)
    c["q"] = (torch.randn(4, 1, 8, 64, generator=g) * 100).to(dtype)
    for h in range(2):
        c["q"][:, :, 4 * h : 4 * h + 4] = c["q"][:, :, 4 * h : 4 * h + 1]      # the rows of a key head alike: one key for all
    for b, pos in enumerate((40, 3, 32, 63)):
        pid = int(c["table"][b, pos // 16])
        c["k_pages"][pid, pos % 16] = c["q"][b, 0].view(2, 4, 64)[:, 0]
        c["v_pages"][pid, pos % 16, :, 9] = float("nan")
    ref, _ = P.paged_attention_reference(**c, dtype=torch.float64)
    d = {x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}
    o = P.paged_attention(**d).cpu()
    dims = [i for i in range(64) if i != 9]
    assert torch.isnan(o[..., 9]).all() and torch.isnan(ref[..., 9]).all()
    assert bool(((o.double() - ref)[..., dims].abs() <= 2.0 ** -20 * ref[..., dims].abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("n,D", [(1, 64), (3, 128)])
def test_a_key_with_an_infinite_component_weighs_nothing(n, D, dt):
    """Its score is -inf for every row; one that is merely far below gives the same bits (no row is summed in another way)."""
    c = att_case(17, [300, 77, 128, 500], n, 16, 8, 4, D, DTYPES[dt], True)
    c["q"] = (c["q"].abs() + 0.1).to(DTYPES[dt])
    out = []
    for low in (-math.inf, -3e4):
        for b, pos in enumerate((20, 70, 127, 450)):
            c["k_pages"][int(c["table"][b, pos // 16]), pos % 16, :, 5] = low
        out.append(P.paged_attention(**{x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}, return_lse=True))
    assert torch.isfinite(out[0][0]).all() and torch.equal(out[0][1], out[1][1])
    assert torch.equal(out[0][0].view(torch.int16), out[1][0].view(torch.int16))


# ---------------------------------------------------------------------------------------------- forward mode
@pytest.mark.parametrize("dev", BINDING)
@pytest.mark.parametrize("why", ["q", "k_pages", "v_pages"])
def test_attention_refuses_tangents(why, dev):
    """Dual tensors of forward-mode differentiation: the result would come back without its tangent.  torch.no_grad() leaves
    forward mode on."""
    c = {"scale": None, "causal": True, **att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True)}
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        c[why] = torch.autograd.forward_ad.make_dual(c[why].cuda() if dev == "cuda" else c[why], torch.ones_like(c[why], device=dev if dev == "cuda" else "cpu"))
        refused_by_the_binding(dev, c, lambda bind, d: bind.paged_attention(
            *(d[x] for x in ("q", "k_pages", "v_pages", "table", "lens", "scale", "causal")), None, False, None, 0, 0))
        if dev == "checks":
            with pytest.raises(ValueError):
                P.paged_attention(**c)


@pytest.mark.parametrize("dev", BINDING)
@pytest.mark.parametrize("why", ["k", "v", "q", "k_pages"])
def test_append_refuses_tangents(why, dev):
    c = {"q": None, "cos": None, "sin": None, "starts": None, "interleaved": False, **_append_args()}
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        c[why] = torch.autograd.forward_ad.make_dual(c[why].cuda() if dev == "cuda" else c[why], torch.ones_like(c[why], device=dev if dev == "cuda" else "cpu"))
        refused_by_the_binding(dev, c, lambda bind, d: bind.paged_append(
            *(d[x] for x in ("k", "v", "k_pages", "v_pages", "table", "lens", "q", "cos", "sin", "starts", "interleaved")), 0))
        if dev == "checks":
            with pytest.raises(ValueError):
                P.paged_append(**c)


@pytest.mark.parametrize("dev", BINDING)
def test_append_refuses_rotation_tables_that_require_a_gradient(dev):
    c = {"q": None, "cos": None, "sin": None, "starts": None, "interleaved": False, **_append_args()}
    c["sin"] = c["sin"].clone().requires_grad_()
    with pytest.raises(ValueError):
        P.paged_append(**c)
    refused_by_the_binding(dev, c, lambda bind, d: bind.paged_append(
        *(d[x] for x in ("k", "v", "k_pages", "v_pages", "table", "lens", "q", "cos", "sin", "starts", "interleaved")), 0))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_one_sequence_of_any_stride(dev):
    """A dimension of one element may have any stride: one sequence, one page, one token, one head."""
    c = att_case(4, [5], 1, 16, 1, 1, 64, torch.bfloat16, True)
    c["k_pages"], c["v_pages"], c["table"] = c["k_pages"][:1], c["v_pages"][:1], torch.zeros(1, 1, dtype=torch.int32)
    c["k_pages"], c["v_pages"] = c["k_pages"].nan_to_num(1.0), c["v_pages"].nan_to_num(1.0, 1.0, 1.0)
    new = torch.randn(2, 1, 1, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    want = {x: y.clone() if torch.is_tensor(y) else y for x, y in c.items()}
    P.paged_append(new[0], new[1], want["k_pages"], want["v_pages"], want["table"], want["lens"])
    ref, _ = P.paged_attention_reference(**want, dtype=torch.float64)

    def odd(x):                                                     # every dimension of one element with a stride of its own
        y = torch.empty_strided(x.shape, [s if n > 1 else 13 + 2 * i for i, (n, s) in enumerate(zip(x.shape, x.stride()))], dtype=x.dtype, device=dev)
        return y.copy_(x)

    d = {x: odd(y) if torch.is_tensor(y) else y for x, y in c.items()}
    P.paged_append(odd(new[0]), odd(new[1]), d["k_pages"], d["v_pages"], d["table"], d["lens"])
    assert torch.equal(d["k_pages"].cpu(), want["k_pages"]) and torch.equal(d["v_pages"].cpu(), want["v_pages"])
    o = P.paged_attention(**d)
    assert bool(((o.cpu().double() - ref).abs() <= att_tolerance(c, ref)).all())


class Undecided:
    def __bool__(self):
        raise TypeError("neither true nor false")


def test_the_device_path_wants_truth_values():
    """A flag that cannot say whether it is true is refused before anything is launched."""
    c = {"scale": None, **att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True)}
    for causal, want in ((Undecided(), False), (True, Undecided())):
        refused_by_the_binding("checks", c, lambda bind, d: bind.paged_attention(
            *(d[x] for x in ("q", "k_pages", "v_pages", "table", "lens", "scale")), causal, None, want, None, 0, 0))
    a = {"q": None, "cos": None, "sin": None, "starts": None, **_append_args()}
    refused_by_the_binding("checks", a, lambda bind, d: bind.paged_append(
        *(d[x] for x in ("k", "v", "k_pages", "v_pages", "table", "lens", "q", "cos", "sin", "starts")), Undecided(), 0))


# ---------------------------------------------------------------------------------------------- every key once
def counting_case(kept, n, page, hq, hkv, D, dt, causal, seed):
    """All scores 0, so a row's weights are 1 / keys seen; dimension d has the value 1024 at one position and 0 elsewhere.  The
    positions lie beside the borders of half tiles, tiles, waves, pages and likely parts, and at both ends."""
    g = torch.Generator().manual_seed(seed)
    need = [max(k, 0) + (n if causal and k >= 0 else 0) for k in kept]
    table, pages = tables(need, page, g)
    kp = torch.randn(pages, page, hkv, D, generator=g).to(dt)
    vp = torch.zeros(pages, page, hkv, D, dtype=dt)
    want = torch.zeros(len(kept), n, hkv, D, dtype=torch.float64)
    for b, m in enumerate(need):
        if m == 0:
            continue
        near = sorted({p for s in (16, 32, 128, page, 1024, m) for x in range(0, m + 1, s) for p in (x - 1, x) if 0 <= p < m})
        ends = near[:4] + near[-n - 4 :]
        pick = torch.randint(0, len(near), (hkv, D), generator=g)
        for h in range(hkv):
            for d in range(D):
                pos = ends[d] if d < len(ends) else near[int(pick[h, d])]
                vp[int(table[b, pos // page]), pos % page, h, d] = 1024.0
                for i in range(n):
                    seen = max(kept[b], 0) + (i + 1 if causal else 0)
                    if pos < seen:
                        want[b, i, h, d] = 1024.0 / seen
    c = dict(q=torch.zeros(len(kept), n, hq, D, dtype=dt), k_pages=kp, v_pages=vp, table=table, lens=torch.tensor(kept, dtype=torch.int32), causal=causal)
    return c, want.repeat_interleave(hq // hkv, 2)


COUNT = [  # kept, n, page, hq, hkv, D, dtype, causal
    ([3001, 0, 127, 128, 2047], 1, 48, 4, 2, 64, "bf16", True),
    ([1500, 777, -1, 16, 5000], 5, 16, 16, 2, 128, "fp16", True),
    ([2900, 33, 4096], 1, 256, 3, 3, 128, "bf16", False),
    ([640, 6001], 40, 64, 2, 2, 64, "fp16", True),
    ([100] * 3 + [9000] + [1] * 30, 3, 32, 12, 2, 64, "bf16", True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(COUNT)))
@pytest.mark.parametrize("share,least", [(None, 0), (0, 0), (1, 1), (7, 3), (64, 1), (700, 1), (256, 1)])
def test_attention_kernel_takes_every_key_once(case, share, least, monkeypatch):
    """A key that is lost shows as 0, one that is taken twice as twice the value.  Weights are equal powers of two and sums of
    them exact; the division and the output each round once.  The log-sum-exp is a logarithm to base 2 below 16 (last place
    2^-20, times ln 2), times an ln 2 that is off by 2^-25 (2^-21 in all), rounded (2^-21): 2^-19 together."""
    kept, n, page, hq, hkv, D, dt, causal = COUNT[case]
    c, want = counting_case(kept, n, page, hq, hkv, D, DTYPES[dt], causal, case)
    monkeypatch.setattr(P, "_DEAL", (share, least))
    o, lse = P.paged_attention(**{x: y.cuda() if torch.is_tensor(y) else y for x, y in c.items()}, return_lse=True)
    err = (o.cpu().double() - want).abs()
    assert bool((err <= (torch.finfo(DTYPES[dt]).eps / 2 + 2.0 ** -21) * want).all()), (err.max(), torch.nonzero(err > 0.01 * want)[:5])
    seen = (torch.tensor(kept).clamp(min=0)[:, None] + (torch.arange(1, n + 1) if causal else torch.zeros(n))) * (torch.tensor(kept) >= 0)[:, None]
    assert bool(((lse.cpu().double() - seen.double().log()[..., None]).nan_to_num(0.0).abs() <= 2.0 ** -19).all())
    assert torch.equal(torch.isneginf(lse.cpu()), (seen == 0)[..., None].expand(lse.shape))


@pytest.mark.parametrize("scale", [2.1e38, -3e38])
def test_attention_refuses_scales_beyond_its_range(scale):
    c = {**att_case(1, [3, 4], 1, 16, 4, 2, 64, torch.bfloat16, True), "scale": scale}
    with pytest.raises(ValueError):
        P.paged_attention(**c)
    refused_by_the_binding("checks", c, lambda bind, d: bind.paged_attention(
        *(d[x] for x in ("q", "k_pages", "v_pages", "table", "lens", "scale", "causal")), None, False, None, 0, 0))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("scale,size", [(1e-36, 1e18), (3e-32, 1e16), (1.9e38, 9e-20), (-1e-36, 1e18), (0.0, 1e14)])
def test_attention_with_scales_at_the_ends_of_their_range(scale, size, dev):
    """q and k are as large or small as it takes for scores of some units."""
    c = att_case(8, [90, 300], 2, 16, 4, 2, 64, torch.bfloat16, True, qscale=0.3)
    c["q"], c["k_pages"] = (c["q"].float() * size).to(torch.bfloat16), (c["k_pages"].float() * size).to(torch.bfloat16)
    d = {x: y.to(dev) if torch.is_tensor(y) else y for x, y in c.items()}
    o, lse = P.paged_attention(**d, scale=scale, return_lse=True)
    ref, ref_lse = P.paged_attention_reference(**c, scale=scale, dtype=torch.float64)
    assert bool((ref_lse.abs() < 64).all())
    assert bool(((o.cpu().double() - ref).abs() <= att_tolerance(c, ref)).all())
    assert bool(((lse.cpu().double() - ref_lse).abs() <= 2.0 ** -24 * 130 * 64).all())


@pytest.mark.gpu
def test_attention_kernel_heads_more_than_2_gb_apart():
    """Heads outside pages and slots, as views of a buffer that holds more than 2^31 bytes of each head."""
    g = torch.Generator().manual_seed(12)
    far, pages, page, hkv, D = (1 << 30) + 8 * 64, 5, 16, 2, 64
    views = []
    for _ in range(2):
        buf = torch.zeros(far + pages * page * D, dtype=torch.bfloat16, device="cuda")
        views.append(buf.as_strided((pages, page, hkv, D), (page * D, D, far, 1)))
    small = [torch.randn(pages, page, hkv, D, generator=g).to(torch.bfloat16) for _ in range(2)]
    for x, y in zip(views, small):
        x.copy_(y)
    table, lens = torch.tensor([[4, 0, 2], [3, 1, -1]], dtype=torch.int32), torch.tensor([40, 20], dtype=torch.int32)
    q = torch.randn(2, 1, 4, D, generator=g).to(torch.bfloat16)
    new = [torch.randn(2, hkv, D, generator=g).to(torch.bfloat16) for _ in range(2)]
    P.paged_append(*(x.cuda() for x in new), *views, table.cuda(), lens.cuda())
    P.paged_append(*new, *small, table, lens)
    assert torch.equal(views[0].cpu(), small[0]) and torch.equal(views[1].cpu(), small[1])
    o = P.paged_attention(q.cuda(), *views, table.cuda(), lens.cuda()).cpu()
    c = dict(q=q, k_pages=small[0], v_pages=small[1], table=table, lens=lens, causal=True)
    ref, _ = P.paged_attention_reference(**c, dtype=torch.float64)
    assert bool(((o.double() - ref).abs() <= att_tolerance(c, ref)).all())
    del views, buf
    torch.cuda.empty_cache()
