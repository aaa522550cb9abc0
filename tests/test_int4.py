"""Linear layers with 4-bit weights, against plain 64-bit products."""
import math

import pytest
import torch

from distributed_llms_amd.ops import int4 as Q

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def layer(seed, n, k, group, zero, sdt):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    codes[0, : min(k, 16)] = torch.arange(16, dtype=torch.uint8)[: min(k, 16)]
    scale = ((torch.rand(n, k // group, generator=g) + 0.1) * (0.3 / math.sqrt(k))).to(sdt)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zero else None
    return codes, scale, z, Q.pack_int4(codes[:, 0::2] | (codes[:, 1::2] << 4), scale, z)


def weights64(codes, scale, z, group):
    zz = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    return (codes.double() - zz) * scale.double().repeat_interleave(group, 1)


def act64(y, act):
    if act == "relu":
        return y.clamp(min=0)
    return 0.5 * y * torch.special.erfc(-y / math.sqrt(2)) if act == "gelu" else y


def check(got, x, codes, scale, z, group, bias, act, res):
    """Tolerance: half a step of the output's type (gelu's slope is at most 1.13), and the fp32 sums.  Codes enter the
    products with an offset of 128 (bf16) or 1024 (fp16) that is taken out again, so a group's sum of |x| (offset + 16) s
    carries up to 16 roundings of 2^-24 (a matrix instruction adds its 32 products in a tree, a group is at most four of
    them, then the offset and the scale); bias, residual and the join of partial sums add a few more of the result."""
    w = weights64(codes, scale, z, group)
    lead = x.shape[:-1]
    x2 = x.double().reshape(-1, x.shape[-1])
    y = x2 @ w.t()
    y = y if bias is None else y + bias.double()
    y = y if res is None else y + res.double().reshape(y.shape)
    ref = act64(y, act)
    off = 128 if x.dtype == torch.bfloat16 else 1024
    mass = x2.abs() @ scale.double().repeat_interleave(group, 1).t()
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + 2.0 ** -24 * (16 * (off + 16) * mass + 64 * y.abs() + 64) * 1.13
    if x.dtype == torch.float16:
        tol += 2.0 ** -25            # below 2^-14 a fp16 step is 2^-24
    assert got.dtype == x.dtype and got.shape == (*lead, codes.shape[0])
    err = (got.double().reshape(y.shape) - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


CASES = [  # rows, n, k, group, zero, act, bias, res, x type, scale type
    (1, 1, 32, 32, False, "none", False, False, "bf16", "bf16"),
    (1, 4096, 1024, 64, False, "gelu", True, False, "bf16", "bf16"),
    (5, 301, 1024, 128, True, "none", True, False, "bf16", "fp16"),
    (16, 33, 96, 32, True, "relu", False, True, "fp16", "fp16"),
    (17, 1000, 448, 64, False, "none", True, True, "fp16", "bf16"),
    (2, 17, 4096, 128, True, "gelu", True, True, "bf16", "bf16"),
    (64, 256, 256, 128, False, "none", False, False, "bf16", "bf16"),
    (65, 130, 160, 32, True, "none", True, False, "bf16", "bf16"),
    (150, 48, 640, 128, False, "relu", True, True, "fp16", "fp16"),
    (3, 5000, 8192, 128, True, "none", True, False, "fp16", "fp16"),
    (40, 777, 2080, 32, True, "gelu", True, True, "bf16", "bf16"),
]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def to(dev, *xs):
    return [None if x is None else x.to(dev) for x in xs]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_matches_plain(dev, i):
    rows, n, k, group, zero, act, has_bias, has_res, dt, sdt = CASES[i]
    codes, scale, z, w = layer(i, n, k, group, zero, DTYPES[sdt])
    g = torch.Generator().manual_seed(50 + i)
    x = torch.randn(rows, k, generator=g).to(DTYPES[dt])
    bias = torch.randn(n, generator=g) if has_bias else None
    res = torch.randn(rows, n, generator=g).to(DTYPES[dt]) if has_res else None
    xd, bd, rd, wd = *to(dev, x, bias, res), w.to(dev)
    got = Q.linear_int4(xd, wd, bd, act=act, res=rd)
    check(got.cpu(), x, codes, scale, z, group, bias, act, res)
    assert torch.equal(Q.linear_int4(xd, wd, bd, act=act, res=rd), got)       # again: the same bits


@pytest.mark.parametrize("dev", DEVICES)
def test_one_feature_at_a_time(dev):
    """x picks single weights: every code of every row comes back from its own place."""
    for k, group in ((160, 32), (256, 128)):
        codes, scale, z, w = layer(k, 50, k, group, True, torch.bfloat16)
        scale.fill_(0.5)
        w.scale.fill_(0.5)
        got = Q.linear_int4(torch.eye(k, dtype=torch.bfloat16).to(dev), w.to(dev)).cpu()
        assert torch.equal(got.double().t(), weights64(codes, scale, z, group))


@pytest.mark.parametrize("dev", DEVICES)
def test_strided_rows_and_leading_dimensions(dev):
    codes, scale, z, w = layer(1, 70, 128, 64, False, torch.bfloat16)
    g = torch.Generator().manual_seed(2)
    big = torch.randn(6, 3, 300, generator=g).to(torch.bfloat16)
    res = torch.randn(6, 3, 90, generator=g).to(torch.bfloat16)
    w = w.to(dev)
    for sl in (slice(0, 128), slice(8, 136), slice(3, 131)):
        x, r = big[..., sl], res[..., 5:75]
        bd, rd = big.to(dev), res.to(dev)
        check(Q.linear_int4(bd[..., sl], w, res=rd[..., 5:75]).cpu(), x, codes, scale, z, 64, None, "none", r)
        check(Q.linear_int4(bd[:, 0, sl], w, res=rd[:, 0, 5:75]).cpu(), x[:, 0], codes, scale, z, 64, None, "none", r[:, 0])
    x = big[0, :, ::2][:, :128]
    check(Q.linear_int4(big.to(dev)[0, :, ::2][:, :128], w).cpu(), x, codes, scale, z, 64, None, "none", None)
    x1 = big[0, 0, :128]
    check(Q.linear_int4(x1.to(dev), w).cpu(), x1, codes, scale, z, 64, None, "none", None)
    assert Q.linear_int4(big[:0, 0, :128].to(dev), w).shape == (0, 70)


@pytest.mark.parametrize("dev", DEVICES)
def test_a_row_with_nan_or_infinity_stays_alone(dev):
    codes, scale, z, w = layer(4, 40, 256, 64, True, torch.bfloat16)
    x = torch.randn(20, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    bad = x.clone()
    bad[3, 7], bad[17, 100] = float("nan"), float("inf")
    got = Q.linear_int4(bad.to(dev), w.to(dev)).cpu()
    assert not torch.isfinite(got[3]).any() and not torch.isfinite(got[17]).all()
    keep = [i for i in range(20) if i not in (3, 17)]
    check(got[keep], x[keep], codes, scale, z, 64, None, "none", None)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", Q.GROUPS)
def test_quantize_is_round_to_nearest(group, symmetric):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(37, 4 * group, generator=g) * 0.05
    w[3, :group] = 0.0
    w[4, :group] = w[4, :group].abs() + 0.1
    q = Q.quantize_int4(w, group, symmetric)
    d = q.dequantize(torch.float64)
    assert torch.equal(d, weights64(q.codes(), q.scale[:, :37].t(), None if q.zero is None else q.zero[:, :37].t(), group))
    s = q.scale[:, :37].t().double().repeat_interleave(group, 1)
    # half a step of the grid; at the ends of the range the stored (bf16) scale and a rounded zero shift it by up to
    # 8 steps 2^-8 + 1/2 step (15 steps 2^-8 + 1/2)
    slack = 8 * 2.0 ** -8 if symmetric else 15 * 2.0 ** -8 + 0.5
    assert bool(((d - w.double()).abs() <= s * (0.5 + slack)).all())
    inside = (q.codes() > 0) & (q.codes() < 15)
    assert bool(((d - w.double()).abs() <= s * 0.5001)[inside].all())
    assert bool((d[3, :group] == 0).all())


REFUSED = {
    "K of another layer": lambda c: c.update(x=c["x"][:, :32]),
    "fp32 rows": lambda c: c.update(x=c["x"].float()),
    "an unknown activation": lambda c: c.update(act="tanh"),
    "bf16 bias": lambda c: c.update(bias=torch.zeros(40, dtype=torch.bfloat16)),
    "short bias": lambda c: c.update(bias=torch.zeros(39)),
    "res of another type": lambda c: c.update(res=torch.zeros(2, 40)),
    "res of another shape": lambda c: c.update(res=torch.zeros(3, 40, dtype=torch.bfloat16)),
}


@pytest.mark.parametrize("why", sorted(REFUSED))
def test_refuses(why):
    c = dict(x=torch.zeros(2, 64, dtype=torch.bfloat16), w=layer(0, 40, 64, 32, False, torch.bfloat16)[3])
    REFUSED[why](c)
    with pytest.raises(ValueError):
        Q.linear_int4(**c)


def test_refuses_to_pack():
    p, s = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 2, dtype=torch.bfloat16)
    Q.pack_int4(p, s)
    for bad in (dict(packed=p.int()), dict(scale=s.float()), dict(scale=torch.ones(4, 3, dtype=torch.bfloat16)), dict(scale=s[:3]),
                dict(zero=torch.zeros(4, 2)), dict(scale=torch.ones(4, 8, dtype=torch.bfloat16)), dict(packed=p[:0], scale=s[:0])):
        with pytest.raises(ValueError):
            Q.pack_int4(**{"packed": p, "scale": s, **bad})
    for bad in (dict(group=48), dict(weight=torch.zeros(4, 100)), dict(weight=torch.zeros(4))):
        with pytest.raises(ValueError):
            Q.quantize_int4(**{"weight": torch.zeros(4, 128), "group": 64, **bad})


MORE_REFUSED = {
    **REFUSED,
    "rows that require a gradient": lambda c: c.update(x=c["x"].clone().requires_grad_()),
    "a bias that requires a gradient": lambda c: c.update(bias=torch.zeros(40, requires_grad=True)),
}


@pytest.mark.parametrize("dev", ["checks", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("why", sorted(set(MORE_REFUSED) - {"an unknown activation"}))
def test_refuses_on_the_device_path(why, dev):
    """The host side for device tensors refuses before it launches, so its checks can be seen without a GPU too."""
    from distributed_llms_amd.ops import _loader

    if dev == "checks" and not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    c = dict(x=torch.zeros(2, 64, dtype=torch.bfloat16), w=layer(0, 40, 64, 32, False, torch.bfloat16)[3], bias=None, res=None)
    MORE_REFUSED[why](c)
    with pytest.raises(ValueError):
        Q.linear_int4(**c)
    to_dev = "cuda" if dev == "cuda" else "cpu"
    (x, bias, res), w = to(to_dev, c["x"], c["bias"], c["res"]), c["w"].to(to_dev)
    with pytest.raises(ValueError):
        _loader.bind().linear_int4(x, w.words, w.scale, w.zero, w.n, w.k, w.group, bias, 0, res, None, 0)


SHAPES = [  # tiles of a wave (None: the wide one of the row count), waves over outputs, waves over K, parts of K
    (1, 1, 8, 1), (1, 2, 4, 3), (1, 4, 2, 64), (None, 1, 4, 1), (None, 2, 2, 2), (None, 1, 4, 5), (None, 1, 1, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("i", [2, 3, 4, 5, 7, 8, 10])
def test_every_launch_shape_is_right(i, shape, monkeypatch):
    """Waves and parts of K that get no features at all included."""
    rows, n, k, group, zero, act, has_bias, has_res, dt, sdt = CASES[i]
    monkeypatch.setattr(Q, "_SHAPE", (shape[0] or (2 if rows <= 16 else 4), *shape[1:]))
    codes, scale, z, w = layer(i, n, k, group, zero, DTYPES[sdt])
    g = torch.Generator().manual_seed(50 + i)
    x = torch.randn(rows, k, generator=g).to(DTYPES[dt])
    bias = torch.randn(n, generator=g) if has_bias else None
    res = torch.randn(rows, n, generator=g).to(DTYPES[dt]) if has_res else None
    xd, bd, rd = to("cuda", x, bias, res)
    check(Q.linear_int4(xd, w.to("cuda"), bd, act=act, res=rd).cpu(), x, codes, scale, z, group, bias, act, res)


@pytest.mark.gpu
def test_rows_too_far_apart_are_gathered():
    """x as every 2^24-th element row of a long buffer."""
    codes, scale, z, w = layer(1, 70, 128, 64, False, torch.bfloat16)
    big = torch.zeros((1 << 24) + 128, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(2, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    rows = big.as_strided((2, 128), (1 << 24, 1))
    rows.copy_(x)
    check(Q.linear_int4(rows, w.to("cuda")).cpu(), x, codes, scale, z, 64, None, "none", None)


def test_quantize_keeps_to_what_scales_can_say():
    w = torch.zeros(3, 64)
    w[0, 5], w[1, 40] = 1e-9, 3.0
    q = Q.quantize_int4(w, 32, scale_dtype=torch.float16)            # 1e-9 / 7 is no fp16 number
    d = q.dequantize()
    assert bool((d[0] == 0).all()) and bool((d[2] == 0).all()) and abs(float(d[1, 40]) - 3.0) <= 3.0 * 2.0 ** -11
    for bad, dt in ((1e7, torch.float16), (math.inf, torch.bfloat16), (math.nan, torch.bfloat16)):
        w[1, 40] = bad
        with pytest.raises(ValueError):
            Q.quantize_int4(w, 32, scale_dtype=dt)


@pytest.mark.parametrize("dev", ["checks", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("change", [dict(n=41 + 16), dict(k=256), dict(group=64), dict(group=0), dict(n=1)], ids=str)
def test_refuses_weights_of_another_layout(change, dev):
    """A layer whose sizes do not fit its words, scales and zeros is refused before it launches."""
    import dataclasses

    from distributed_llms_amd.ops import _loader

    if dev == "checks" and not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    w = dataclasses.replace(layer(0, 40, 128, 32, True, torch.bfloat16)[3].to("cuda" if dev == "cuda" else "cpu"), **change)
    x = torch.zeros(2, w.k, dtype=torch.bfloat16, device=w.words.device)
    with pytest.raises(ValueError):
        _loader.bind().linear_int4(x, w.words, w.scale, w.zero, w.n, w.k, w.group, None, 0, None, None, 0)


BY_RULE = [  # rows, n, k, group, zero, res: sizes at which the rule's shapes differ, with odd ends of outputs and features
    (24, 4203, 1024, 64, True, True), (33, 4100, 960, 64, False, False), (70, 2101, 2048, 128, True, False), (24, 1024, 4064, 32, True, True),
    (16, 4201, 512, 32, False, True), (9, 12301, 288, 32, True, False), (200, 1030, 1152, 128, False, True), (17, 16400, 256, 128, True, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(BY_RULE)))
def test_shapes_of_the_rule(i):
    rows, n, k, group, zero, has_res = BY_RULE[i]
    dt, sdt = (torch.float16, torch.bfloat16) if i % 2 else (torch.bfloat16, torch.float16)
    codes, scale, z, w = layer(90 + i, n, k, group, zero, sdt)
    g = torch.Generator().manual_seed(190 + i)
    x = torch.randn(rows, k, generator=g).to(dt)
    res = torch.randn(rows, n, generator=g).to(dt) if has_res else None
    xd, rd = to("cuda", x, res)
    check(Q.linear_int4(xd, w.to("cuda"), res=rd).cpu(), x, codes, scale, z, group, None, "none", res)


# ---------------------------------------------------------------------------------------------- odd rows
def odd_rows(dt, k):
    """Rows with infinities and NaN, and, in bf16, near the end of the type's range; one ordinary row behind them."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(7, k, generator=g)
    x[0, 3], x[1, k - 1] = math.inf, -math.inf
    x[2, 0], x[2, k // 2] = math.inf, math.inf
    x[3, 40] = math.nan
    big = 3e38 if dt == torch.bfloat16 else 6e4
    x[4, 5], x[4, 90], x[5, 50] = big, -big, big
    return x.to(dt)


def check_odd(got, x, codes, scale, z, group, act="none"):
    """Infinities and NaN where the formula has them (a weight of 0 times infinity among them); elsewhere half a step, 2^-14
    of the sum of |x w| for sums of up to 1000 products in fp32, and the codes' offset as in ``check``: an output whose weights
    are all 0 is the difference of two sums of 16 to 31 |x|, each with 16 roundings of 2^-24."""
    w = weights64(codes, scale, z, group)
    y = x.double() @ w.t()
    ref = act64(y, act)
    top = torch.finfo(x.dtype).max
    assert bool((ref.abs() < top)[torch.isfinite(ref)].all())
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isposinf(got), torch.isposinf(ref))
    assert torch.equal(torch.isneginf(got), torch.isneginf(ref))
    ok = torch.isfinite(ref)
    mass = x.double().abs().nan_to_num(0, 0, 0)
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + 2.0 ** -14 * (mass @ w.abs().t()) + 2.0 ** -24
    tol += 2.0 ** -24 * 16 * 32 * (mass @ scale.double().repeat_interleave(group, 1).t())
    assert bool(((got.double() - ref).abs()[ok] <= tol[ok]).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("k,group,shape", [(256, 64, None), (160, 32, None), (640, 128, (1, 1, 4, 3)), (640, 64, (1, 2, 2, 1))])
def test_infinite_and_largest_rows(k, group, shape, zero, dt, dev, monkeypatch):
    monkeypatch.setattr(Q, "_SHAPE", shape)
    codes, scale, z, w = layer(8, 83, k, group, zero, torch.bfloat16)
    codes[:4] = 8 if z is None else z[:4].repeat_interleave(group, 1)           # outputs whose weights are all 0
    w = Q.pack_int4(codes[:, 0::2] | (codes[:, 1::2] << 4), scale, z)
    x = odd_rows(DTYPES[dt], k)
    check_odd(Q.linear_int4(x.to(dev), w.to(dev)).cpu(), x, codes, scale, z, group)
    more = torch.cat((x, x, x))                                                  # the kernels for more than 16 rows
    if shape is None:
        check_odd(Q.linear_int4(more.to(dev), w.to(dev)).cpu(), more, codes, scale, z, group)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("act", ["relu", "gelu"])
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_nan_stays_nan_behind_an_activation(dt, act, dev):
    codes, scale, z, w = layer(8, 40, 128, 64, False, torch.bfloat16)
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(2)).to(DTYPES[dt])
    x[2, 17] = math.nan
    bias = torch.zeros(40)
    bias[9] = math.nan
    got = Q.linear_int4(x.to(dev), w.to(dev), bias.to(dev), act=act).cpu()
    want = torch.zeros(4, 40, dtype=torch.bool)
    want[2], want[:, 9] = True, True
    assert torch.equal(torch.isnan(got), want)


# ---------------------------------------------------------------------------------------------- bits of the sums
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("k,group", [(1024, 64), (8192, 128), (4096, 32)])
def test_sums_keep_32_bits(k, group, dt, dev):
    """Rows of positive numbers (behind relu), whose sum is far larger than the output: what a code is shifted by on its way into
    the products must not eat the sum's bits.  The bias is the negated result, so the output is the error, in fine steps.
    A group of q = G / 32 matrix instructions has at most 8 q full-size roundings in each of its two sums of up to 31 sum |x|,
    spread evenly over half a step of 2^-24: sqrt(16 q / 12) 31 2^-24 s sum |x| per group, added up over groups as independent
    errors are, and the output's own sum (a rounding of 2^-24 of it per group, and the bias)."""
    codes, scale, z, w = layer(3, 600, k, group, False, torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    x = (torch.rand(6, k, generator=g) + 0.5).to(DTYPES[dt])
    big = scale * 64                                             # errors well above the output type's last step
    w = Q.pack_int4(codes[:, 0::2] | (codes[:, 1::2] << 4), big).to(dev)
    ref = x.double() @ weights64(codes, big, None, group).t()
    mass = x.double().view(6, 1, k // group, group).sum(-1) * big.double()             # [6, 600, groups]
    bound = math.sqrt(16 * (group // 32) / 12) * 31 * 2.0 ** -24 * mass.pow(2).sum(-1).sqrt()
    bound = bound + 2.0 ** -24 * math.sqrt(k // group + 2) * ref.abs().amax()
    err = torch.stack([Q.linear_int4(x[i : i + 1].to(dev), w, -ref[i].float().to(dev)).cpu().double()[0] - (ref[i] - ref[i].float().double())
                       for i in range(6)])
    rms, most = float((err / bound).pow(2).mean().sqrt()), float((err / bound).abs().max())
    assert rms <= 1.0 and most <= 6.0, (rms, most)                # 3600 outputs: six standard deviations


@pytest.mark.parametrize("dev", ["checks", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("why", ["x", "bias", "res"])
def test_refuses_tangents(why, dev):
    """Dual tensors of forward-mode differentiation: the result would come back without its tangent."""
    from distributed_llms_amd.ops import _loader

    if dev == "checks" and not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    at = "cuda" if dev == "cuda" else "cpu"
    c = dict(x=torch.zeros(2, 64, dtype=torch.bfloat16, device=at), bias=torch.zeros(40, device=at), res=torch.zeros(2, 40, dtype=torch.bfloat16, device=at))
    w = layer(0, 40, 64, 32, False, torch.bfloat16)[3].to(at)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        c[why] = torch.autograd.forward_ad.make_dual(c[why], torch.ones_like(c[why]))
        with pytest.raises(ValueError):
            Q.linear_int4(c["x"], w, c["bias"], res=c["res"])
        with pytest.raises(ValueError):
            _loader.bind().linear_int4(c["x"], w.words, w.scale, w.zero, w.n, w.k, w.group, c["bias"], 0, c["res"], None, 0)


@pytest.mark.parametrize("dev", ["checks", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refuses_scales_that_require_a_gradient(dev):
    from distributed_llms_amd.ops import _loader

    if dev == "checks" and not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    at = "cuda" if dev == "cuda" else "cpu"
    x, scale = torch.zeros(2, 64, dtype=torch.bfloat16, device=at), torch.ones(40, 2, dtype=torch.bfloat16, device=at, requires_grad=True)
    w = Q.pack_int4(torch.zeros(40, 32, dtype=torch.uint8, device=at), scale)
    with pytest.raises(ValueError):
        Q.linear_int4(x, w)
    with pytest.raises(ValueError):
        _loader.bind().linear_int4(x, w.words, w.scale, w.zero, w.n, w.k, w.group, None, 0, None, None, 0)
    with torch.no_grad():
        assert Q.linear_int4(x, w).shape == (2, 40)


@pytest.mark.parametrize("dev", DEVICES)
def test_one_output_and_one_row_of_any_stride(dev):
    codes, scale, z, w = layer(5, 1, 64, 32, False, torch.bfloat16)
    x = torch.randn(1, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    bias, res = torch.randn(3, generator=torch.Generator().manual_seed(3))[::3], torch.ones(1, 7, dtype=torch.bfloat16)[:, ::7]
    assert bias.stride() == (3,) and res.stride(1) == 7
    xd = torch.empty_strided((1, 64), (13, 1), dtype=torch.bfloat16, device=dev).copy_(x)
    bd = torch.empty_strided((1,), (3,), device=dev).copy_(bias)
    rd = torch.empty_strided((1, 1), (7, 7), dtype=torch.bfloat16, device=dev).copy_(res)
    check(Q.linear_int4(xd, w.to(dev), bd, res=rd).cpu(), x, codes, scale, z, 32, bias, "none", res)
