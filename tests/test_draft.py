"""Verification of drafted tokens: whole numbers, compared exactly with a plain implementation in 64 bits."""
import pytest
import torch

from distributed_llms_amd.ops.draft import verify_draft

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def plain(draft, target, u, proposal=None, counts=None, pad=-1):
    """All sequences at once, in 64 bits (independent of the oracle's loop)."""
    B, n = draft.shape
    V = target.shape[2]
    p, uu, x = target.double(), u.double().nan_to_num(0.0), draft.long()
    q = proposal.double() if proposal is not None else torch.zeros(B, n, V, dtype=torch.float64)
    valid = (x >= 0) & (x < V)
    if proposal is None and n:
        q.scatter_(2, x.clamp(0, V - 1)[..., None], valid.double()[..., None])
    c = torch.full((B,), n) if counts is None else counts.long().clamp(0, n)
    at = x.clamp(0, V - 1)[..., None]
    ok = valid & (uu[:, :n] * q.gather(2, at)[..., 0] < p[:, :n].gather(2, at)[..., 0]) & (torch.arange(n) < c[:, None])
    acc = ok.long().cumprod(1).sum(1)
    q = torch.cat((q, torch.zeros(B, 1, V, dtype=torch.float64)), 1)
    b = torch.arange(B)
    row = p[b, acc]
    w = (row - q[b, acc] * (acc < c)[:, None])
    w = torch.where(w > 0, w, 0.0)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, torch.where(row > 0, row, 0.0))
    F = w.cumsum(1)
    at = (F > uu[:, n:].clamp(0, 1) * F[:, -1:]) & (w > 0)
    last = V - 1 - (w > 0).flip(1).long().argmax(1)
    hit = torch.where(at.any(1), at.long().argmax(1), last)
    hit = torch.where((F[:, -1] > 0) & torch.isfinite(F[:, -1]), hit, 0)
    j = torch.arange(n + 1)
    full = torch.cat((x, torch.zeros(B, 1, dtype=torch.long)), 1)
    tokens = torch.where(j < acc[:, None], full, torch.where(j == acc[:, None], hit[:, None], pad))
    return tokens.to(torch.int32), acc.to(torch.int32)


def case(seed, B, n, V, dt, proposal=True, ragged=True, noise=0.4):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, n + 1, V, generator=g) * 2
    prop = logits[:, :n] + torch.randn(B, n, V, generator=g) * noise
    e = torch.empty(B, n, V).exponential_(generator=g)
    draft = (prop - e.log()).argmax(-1).to(torch.int32) if n else torch.zeros(B, 0, dtype=torch.int32)
    return dict(draft=draft, target=logits.softmax(-1).to(dt), u=torch.rand(B, n + 1, generator=g),
                proposal=prop.softmax(-1).to(dt) if proposal else None,
                counts=torch.randint(0, n + 1, (B,), generator=g).to(torch.int32) if ragged else None)


def same(got, want):
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0]), (got, want)


def on(c, dev):
    return {k: v.to(dev) if torch.is_tensor(v) else v for k, v in c.items()}


CASES = [  # B, n, V, dtype, proposal, ragged
    (1, 0, 1, "fp32", False, False), (1, 4, 50265, "fp32", True, False), (3, 1, 2, "bf16", True, True),
    (7, 7, 272, "fp32", True, True), (5, 3, 1000, "fp16", False, True), (64, 5, 4097, "bf16", True, False),
    (2, 63, 97, "fp32", True, True), (2, 2, 151937, "fp32", False, False), (300, 1, 65, "fp32", True, True),
    (4, 3, 30011, "bf16", True, False), (40, 0, 777, "fp16", False, False),
    (130, 2, 9001, "fp16", True, True), (3, 2, 8192, "fp32", True, True), (3, 2, 8193, "bf16", False, True), (5, 2, 1024, "fp32", True, True),
    (2, 1, 1025, "fp32", True, True), (33, 2, 20011, "fp32", True, True),
]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("k", range(len(CASES)))
def test_matches_plain(dev, k):
    B, n, V, dt, proposal, ragged = CASES[k]
    for seed in range(3):
        c = case(100 * k + seed, B, n, V, DTYPES[dt], proposal, ragged)
        same(verify_draft(**on(c, dev)), plain(**c))


@pytest.mark.parametrize("dev", DEVICES)
def test_borders(dev):
    """Probabilities that are multiples of 1 / 8: every sum is exact, so borders are hit exactly."""
    p = torch.tensor([0, 1, 0, 3, 0, 0, 4, 0], dtype=torch.float32) / 8
    for u, want in ((0.0, 1), (0.124, 1), (0.125, 3), (0.499, 3), (0.5, 6), (0.999, 6), (1.0, 6), (-1.0, 1), (float("nan"), 1)):
        c = dict(draft=torch.zeros(1, 0, dtype=torch.int32), target=p.view(1, 1, 8), u=torch.tensor([[u]]))
        got = verify_draft(**on(c, dev))
        assert int(got[0]) == want and int(got[1]) == 0, u
    # acceptance is strict: u q < p
    q = torch.tensor([0, 2, 0, 3, 0, 0, 3, 0], dtype=torch.float32) / 8
    for u, accepted in ((0.5, 0), (0.4999, 1)):
        c = dict(draft=torch.tensor([[1]], dtype=torch.int32), target=p.expand(1, 2, 8).contiguous(), u=torch.tensor([[u, 0.99]]),
                 proposal=q.view(1, 1, 8))
        got = verify_draft(**on(c, dev))
        assert int(got[1]) == accepted and got[0].tolist() == ([[1, 6]] if accepted else [[6, -1]])
        same(got, plain(**c))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_odd_rows(dev, dt):
    """Drafts outside the vocabulary, a target below its proposal everywhere, rows without weight, with NaN, with infinity."""
    B, n, V = 8, 3, 300
    c = case(7, B, n, V, DTYPES[dt], ragged=False)
    c["draft"][0, 0], c["draft"][1, 1], c["draft"][2, 2] = V, -1, 1 << 30
    c["target"][3, 0] = c["proposal"][3, 0] * 0.25
    c["u"][3, 0] = 0.9
    c["target"][4] = 0
    c["target"][5] = float("nan")
    c["target"][6, :, 5] = float("inf")
    c["proposal"][7] = 0
    c["counts"] = torch.tensor([3, 3, 3, 3, 3, 3, -4, 99], dtype=torch.int32)
    want = plain(**c)
    got = verify_draft(**on(c, dev), pad=-1)
    same(got, want)
    assert int(want[0][4, 0]) == 0 and int(want[0][5, 0]) == 0 and int(want[0][6, 0]) == 0
    c["proposal"] = None
    same(verify_draft(**on(c, dev)), plain(**c))


@pytest.mark.parametrize("dev", DEVICES)
def test_strided_rows(dev):
    """Rows of padded logits, one step of a longer buffer, an odd row stride and an odd first element."""
    for off in (0, 1, 3):
        c = case(9, 5, 4, 1001, torch.float32)
        d = on(c, dev)
        for name, rows in (("target", 5), ("proposal", 4)):
            big = torch.full((5, rows + 2, 1001 + 14 + off), float("nan"), device=dev)
            big[:, 1 : rows + 1, off : off + 1001] = d[name]
            d[name] = big[:, 1 : rows + 1, off : off + 1001]
        d["u"] = torch.cat((d["u"], d["u"]), 1)[:, :5]
        d["draft"] = torch.cat((d["draft"], d["draft"]), 1)[:, :4]
        same(verify_draft(**d), plain(**c))


@pytest.mark.parametrize("dev", DEVICES)
def test_distribution_is_the_targets(dev):
    """20 000 sequences: the first kept token follows the target whatever the proposal.  Its frequencies are sums of
    independent draws with variance p (1 - p) / N < 1.25e-5 / N * 1e4; five standard deviations bound each of them."""
    N, V = 20000, 12
    g = torch.Generator().manual_seed(3)
    p, q = (torch.randn(V, generator=g).softmax(-1) for _ in range(2))
    draft = torch.multinomial(q, N, replacement=True, generator=g).to(torch.int32)[:, None]
    c = dict(draft=draft, target=p.expand(N, 2, V).contiguous(), u=torch.rand(N, 2, generator=g), proposal=q.expand(N, 1, V).contiguous())
    if dev == "cpu":
        tokens = plain(**c)[0]
    else:
        tokens = verify_draft(**on(c, dev))[0].cpu()
    freq = torch.bincount(tokens[:, 0].long(), minlength=V).double() / N
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / N).sqrt()).all())


REFUSED = {
    "64-bit draft": lambda c: c.update(draft=c["draft"].long()),
    "one row too few": lambda c: c.update(target=c["target"][:, :3]),
    "proposal of another type": lambda c: c.update(proposal=c["proposal"].half()),
    "proposal of another vocabulary": lambda c: c.update(proposal=c["proposal"][..., :9]),
    "u too short": lambda c: c.update(u=c["u"][:, :3]),
    "64-bit u": lambda c: c.update(u=c["u"].double()),
    "counts of another batch": lambda c: c.update(counts=c["counts"][:1]),
    "64-bit target": lambda c: c.update(target=c["target"].double()),
    "vocabulary strided": lambda c: c.update(target=c["target"].transpose(1, 2).contiguous().transpose(1, 2)),
    "64 drafts": lambda c: c.update(case(0, 2, 64, 10, torch.float32)),
}


@pytest.mark.parametrize("why", sorted(REFUSED))
def test_refuses(why):
    c = case(1, 2, 3, 10, torch.float32)
    REFUSED[why](c)
    with pytest.raises(ValueError):
        verify_draft(**c)


@pytest.mark.parametrize("dev", ["checks", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("why", sorted(REFUSED))
def test_refuses_on_the_device_path(why, dev):
    """The host side for device tensors refuses before it launches, so its checks can be seen without a GPU too."""
    from distributed_llms_amd.ops import _loader

    if dev == "checks" and not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    c = case(1, 2, 3, 10, torch.float32)
    REFUSED[why](c)
    d = on(c, "cuda" if dev == "cuda" else "cpu")
    args = [d[x] for x in ("draft", "target", "u", "proposal", "counts")]
    with pytest.raises(ValueError):
        _loader.bind().verify_draft(*args, -1, None, 0)
    with pytest.raises(ValueError):
        _loader.bind().verify_draft(*args, 1 << 40, None, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("pieces", [1, 2, 7, 48, 64])
@pytest.mark.parametrize("k", [2, 4, 5, 6, 9, 11, 13, 16])
def test_rows_in_pieces(k, pieces, monkeypatch):
    """Any number of pieces, also more than there are tokens."""
    from distributed_llms_amd.ops import draft as D

    monkeypatch.setattr(D, "_PIECES", pieces)
    B, n, V, dt, proposal, ragged = CASES[k]
    c = case(100 * k, min(B, 40), n, V, DTYPES[dt], proposal, ragged)
    same(verify_draft(**on(c, "cuda")), plain(**c))


@pytest.mark.gpu
@pytest.mark.parametrize("pieces", [1, 2, 7, 48, 64])
@pytest.mark.parametrize("V", [64, 700, 5000, 12000])
def test_the_last_token_stands_for_the_end_of_the_row(V, pieces, monkeypatch):
    """u = 1: no cumulative weight lies beyond it, so the last token with weight is the answer whatever the sums' rounding;
    weights end at another token in every sequence."""
    from distributed_llms_amd.ops import draft as D

    monkeypatch.setattr(D, "_PIECES", pieces)
    g = torch.Generator().manual_seed(V)
    p = torch.rand(60, 1, V, generator=g) + 1e-3
    last = torch.randint(0, V, (60,), generator=g)
    p[torch.arange(V)[None, None] > last[:, None, None]] = 0.0
    tokens, accepted = verify_draft(torch.zeros(60, 0, dtype=torch.int32, device="cuda"), p.cuda(), torch.ones(60, 1, device="cuda"))
    assert torch.equal(tokens.cpu()[:, 0].long(), last) and not bool(accepted.any())


@pytest.mark.parametrize("dev", DEVICES)
def test_one_draft_of_any_stride(dev):
    """A dimension of one element may have any stride: one draft, one number, one count taken out of larger tensors."""
    strided = lambda x, *st: torch.empty_strided(x.shape, st, dtype=x.dtype, device=dev).copy_(x)  # noqa: E731
    c = case(3, 6, 1, 700, torch.float32)
    same(verify_draft(**{**on(c, dev), "draft": strided(c["draft"], 1, 6)}), plain(**c))
    c = case(4, 1, 0, 700, torch.float32)
    same(verify_draft(**{**on(c, dev), "u": strided(c["u"], 9, 5), "counts": strided(c["counts"], 3)}), plain(**c))
    c = case(5, 4, 2, 1, torch.float32)
    d = {**on(c, dev), "target": strided(c["target"], 12, 3, 2), "proposal": strided(c["proposal"], 12, 3, 2)}
    same(verify_draft(**d), plain(**c))


def test_distribution_is_the_targets_on_the_cpu():
    """As above, through the operator itself: five standard deviations of 3000 draws."""
    N, V = 3000, 6
    g = torch.Generator().manual_seed(8)
    p, q = (torch.randn(V, generator=g).softmax(-1) for _ in range(2))
    draft = torch.multinomial(q, N, replacement=True, generator=g).to(torch.int32)[:, None]
    tokens, accepted = verify_draft(draft, p.expand(N, 2, V), torch.rand(N, 2, generator=g), proposal=q.expand(N, 1, V))
    freq = torch.bincount(tokens[:, 0].long(), minlength=V).double() / N
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / N).sqrt()).all())
    rate = torch.minimum(p, q).sum()                                          # of accepted drafts
    assert abs(float(accepted.double().mean() - rate)) <= 5 * float((rate * (1 - rate) / N).sqrt())
