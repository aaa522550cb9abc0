"""The decode-step operators together (append, attention, 4-bit layers, verification), captured and on several streams, and
in the transformer recognizer: decoders longer than 1024 positions, images of more than 1024 patches, 4-bit weights."""
import dataclasses
import math
import random

import pytest
import torch

from distributed_llms_amd.models.trocr import TrOCR, TrOCRConfig
from distributed_llms_amd.ops import _loader
from distributed_llms_amd.ops import draft as D
from distributed_llms_amd.ops import int4 as Q
from distributed_llms_amd.ops import paged as P

HQ, HKV, DIM, PAGE, VOCAB, N = 8, 2, 64, 16, 300, 4
HID = HQ * DIM


class Layer:
    """One attention layer between an embedding and a vocabulary projection, all linears 4-bit."""

    def __init__(self, dev, B, seed=0, width=12):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.B, self.dev = B, dev
        self.tok = r(VOCAB, HID).to(torch.bfloat16).to(dev)
        self.qkv = Q.quantize_int4(r((HQ + 2 * HKV) * DIM, HID) * 0.06, 64, symmetric=False).to(dev)
        self.out = Q.quantize_int4(r(HID, HID) * 0.05, 128).to(dev)
        self.head = Q.quantize_int4(r(VOCAB, HID) * 0.08, 64).to(dev)
        self.bias = r(VOCAB).to(dev)
        self.cos, self.sin = P.rope_tables(width * PAGE, 32, device=dev)
        self.k, self.v = (torch.full((B * width, PAGE, HKV, DIM), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
        self.table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).to(dev)
        self.lens = torch.tensor([0, 7, 60, 130, -1, 15][:B], dtype=torch.int32, device=dev)
        self.table[self.lens < 0] = -1
        for b, n in enumerate(self.lens.tolist()):              # what the sequences kept before
            if n > 0:
                k, v = (r(n, HKV, DIM).to(torch.bfloat16).to(dev) for _ in range(2))
                one = torch.zeros(1, dtype=torch.int32, device=dev)
                P.paged_append(k, v, self.k, self.v, self.table[b : b + 1], one, starts=torch.tensor([0, n], dtype=torch.int32, device=dev))
        self.last = torch.randint(0, VOCAB, (B, 1), generator=g, dtype=torch.int32).to(dev)

    def target(self, draft):
        """Probabilities of the target behind [last, draft]: [B, N + 1, VOCAB] fp32, and what is on the way."""
        B, tokens = self.B, torch.cat((self.last, draft), 1)
        x = self.tok[tokens.long()]
        qkv = Q.linear_int4(x, self.qkv).view(B * (N + 1), HQ + 2 * HKV, DIM)
        q, k, v = qkv[:, :HQ], qkv[:, HQ : HQ + HKV], qkv[:, HQ + HKV :]
        qr = P.paged_append(k, v, self.k, self.v, self.table, self.lens, q=q, cos=self.cos, sin=self.sin, interleaved=True)
        a = P.paged_attention(qr.view(B, N + 1, HQ, DIM), self.k, self.v, self.table, self.lens)
        h = Q.linear_int4(a.reshape(B, N + 1, HID), self.out, res=x)
        logits = Q.linear_int4(h, self.head, self.bias)
        return torch.softmax(logits.float(), -1), (x, qkv, qr, a, h, logits)

    def step(self, draft, u, proposal):
        p, _ = self.target(draft)
        tokens, accepted = D.verify_draft(draft, p, u, proposal=proposal)
        self.last.copy_(tokens.gather(1, accepted.long()[:, None]))
        self.lens.add_(torch.where(self.lens >= 0, accepted + 1, torch.zeros_like(accepted)))
        return tokens, accepted


def drafts(seed, B):
    g = torch.Generator().manual_seed(seed)
    prop = torch.softmax(torch.randn(B, N, VOCAB, generator=g) * 2, -1)
    draft = torch.multinomial(prop.view(-1, VOCAB), 1, generator=g).view(B, N).to(torch.int32)
    return draft, torch.rand(B, N + 1, generator=g), prop


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
def test_a_decode_step_stage_by_stage(dev):
    """Every stage against 64 bits on the inputs it got, over four steps whose lengths follow the verification."""
    B = 6
    m = Layer(dev, B)
    for step in range(4):
        draft, u, prop = drafts(step, B)
        k0, v0, lens = m.k.cpu().clone(), m.v.cpu().clone(), m.lens.cpu().clone()
        p, (x, qkv, qr, a, h, logits) = m.target(draft.to(dev))
        c = lambda t: t.detach().cpu()  # noqa: E731

        def close(got, ref, slack):
            err = (c(got).double() - ref).abs()
            assert bool((err <= 2.0 ** -8 * ref.abs() + slack).all()), float(err.max())

        close(qkv.view(B, N + 1, -1), c(x).double() @ m.qkv.to("cpu").dequantize(torch.float64).t(), 2e-3)
        # the cache and the rotated queries: the oracle's maths on 64-bit tables
        q, k, v = (c(t) for t in (qkv[:, :HQ], qkv[:, HQ : HQ + HKV], qkv[:, HQ + HKV :]))
        kd, vd = k0.double(), v0.double()
        qd = P.paged_append_reference(k.double(), v.double(), kd, vd, c(m.table), lens, q.double(), c(m.cos).double(), c(m.sin).double(),
                                      interleaved=True)
        close(qr, qd, 1e-5)
        seen = ~torch.isnan(kd)
        assert torch.equal(seen, ~torch.isnan(c(m.k)))
        close(m.k[seen.to(dev)], kd[seen], 1e-5)
        assert torch.equal(c(m.v).double().nan_to_num(7.0), vd.nan_to_num(7.0))
        ref, _ = P.paged_attention_reference(c(qr).view(B, N + 1, HQ, DIM), c(m.k), c(m.v), c(m.table), lens, dtype=torch.float64)
        close(a, ref, 1e-3)
        assert bool((a[lens < 0] == 0).all())
        close(h, c(a).double().reshape(B, N + 1, HID) @ m.out.to("cpu").dequantize(torch.float64).t() + c(x).double(), 2e-3)
        close(logits, c(h).double() @ m.head.to("cpu").dequantize(torch.float64).t() + c(m.bias).double(), 4e-3)
        got = D.verify_draft(draft.to(dev), p, u.to(dev), proposal=prop.to(dev))
        want = D.verify_draft_reference(draft, c(p), u, prop)
        assert torch.equal(c(got[0]), want[0]) and torch.equal(c(got[1]), want[1])
        m.last.copy_(got[0].gather(1, got[1].long()[:, None]))
        m.lens.add_(torch.where(m.lens >= 0, got[1] + 1, torch.zeros_like(got[1])))
    assert int(m.lens[4]) == -1 and bool((c(m.lens)[[0, 1, 2, 3, 5]] >= torch.tensor([4, 11, 64, 134, 19])).all())


@pytest.mark.gpu
def test_a_captured_step_follows_the_lengths():
    """One capture, many replays: the lengths advance on the device, eager work and synchronizations in between.  Every replay
    gives the bits of an eager step on a second state."""
    B = 6
    m, e = Layer("cuda", B), Layer("cuda", B)
    draft, u, prop = (x.cuda() for x in drafts(0, B))
    keep = {n: getattr(m, n).clone() for n in ("k", "v", "lens", "last")}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.step(draft, u, prop)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = m.step(draft, u, prop)
    for n, t in keep.items():
        getattr(m, n).copy_(t)
    for i in range(6):
        d, uu, pr = drafts(10 + i, B)
        draft.copy_(d)
        u.copy_(uu)
        prop.copy_(pr)
        graph.replay()
        want = e.step(d.cuda(), uu.cuda(), pr.cuda())
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
        assert torch.equal(m.lens, e.lens) and torch.equal(m.last, e.last)
        assert torch.equal(m.k.view(torch.int16), e.k.view(torch.int16)) and torch.equal(m.v.view(torch.int16), e.v.view(torch.int16))


@pytest.mark.gpu
def test_two_streams_at_once():
    """Two states stepped in turn on two streams of their own, nothing waiting in between: as if each were alone.  Long caches
    and a large vocabulary, so that every workspace (parts of sequences, of K, of rows) is in use on both."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    w = Q.quantize_int4(torch.randn(9000, 8192, generator=g).cuda() * 0.01, 128)
    sets = []
    for _ in range(2):
        kp, vp = r(130, 64, 2, 128), r(130, 64, 2, 128)
        sets.append(dict(q=r(2, 3, 16, 128), k=kp, v=vp, table=torch.randperm(130, generator=g)[:128].view(2, 64).to(torch.int32).cuda(),
                         lens=torch.tensor([4000, 1500], dtype=torch.int32).cuda(), x=r(20, 8192),
                         draft=torch.randint(0, 40000, (3, 2), generator=g).to(torch.int32).cuda(),
                         p=torch.softmax(torch.randn(3, 3, 40000, generator=g).cuda(), -1), u=torch.rand(3, 3, generator=g).cuda() * 1e-4))

    def work(s):
        o, lse = P.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], return_lse=True)
        y = Q.linear_int4(s["x"], w)
        return (o, lse, y, *D.verify_draft(s["draft"], s["p"], s["u"]))

    rules = _loader.bind()
    assert rules.rule_shape(20, 9000, 8192)[3] > 1 and rules.rule_deal(4, 24, 4096, 128)[0] and rules.rule_pieces(3, 40000) > 1
    alone = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(work(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, alone[i]))


# ---------------------------------------------------------------------------------------------- in the recognizer
SMALL = TrOCRConfig(image_size=64, patch=16, enc_dim=128, enc_layers=2, enc_heads=2, enc_mlp=256, dec_dim=128,
                    dec_layers=2, dec_heads=2, dec_ffn=256, vocab=300, max_len=12)


def model(cfg, seed=0):
    torch.manual_seed(seed)
    m = TrOCR(cfg).eval()
    with torch.no_grad():                      # decisive logits: bf16 rounding does not choose the token
        m.lm_head.weight.mul_(8.0)
        m.tok.weight.mul_(4.0)
        m.pos.weight.mul_(4.0)
    return m


def image(cfg, B, dev):
    x = torch.randn(B, 3, cfg.image_size, cfg.image_size, generator=torch.Generator().manual_seed(5))
    y = torch.zeros(B, cfg.image_size, cfg.image_size, 8, dtype=torch.bfloat16)
    y[..., :3] = x.permute(0, 2, 3, 1).to(torch.bfloat16)
    return x, y.to(dev)


def check_tokens(ref, x, toks):
    """Teacher-force the PyTorch model on the produced tokens: nearly every one is (nearly) its own choice."""
    toks = toks.cpu().long()
    with torch.no_grad():
        prefix = torch.cat([torch.full((toks.shape[0], 1), ref.cfg.bos, dtype=torch.long), toks[:, :-1]], 1)
        logits = ref.decode_logits_reference(ref.encode_reference(x), prefix)
    gap = logits.max(-1).values - logits.gather(-1, toks[..., None])[..., 0]
    near = gap < 0.15 * logits.std()
    assert near.float().mean().item() > 0.9, near.float().mean()
    return near


@pytest.mark.gpu
def test_recognizer_beyond_1024_positions():
    cfg = dataclasses.replace(SMALL, max_len=1100)
    ref = model(cfg)
    x, xin = image(cfg, 3, "cuda")
    m = model(cfg).cuda().prepare()
    toks, conf = m.generate(xin, eos_check_every=0)
    assert toks.shape == (3, 1100) and torch.isfinite(conf).all()
    st = next(iter(m._graphs.values())).state
    assert st.lens is not None and int(st.lens[0]) == 1100
    live = (toks != cfg.pad).long().cumprod(1).sum(1)          # behind its eos a sequence is not recorded
    n = max(1, int(live.min()))
    near = check_tokens(ref, x, toks[:, :n])
    if n > 1024:
        assert near[:, 1024:].float().mean().item() > 0.9
    eager, _ = m.generate(xin, max_len=40, use_graph=False, eos_check_every=0)
    assert torch.equal(eager, toks[:, :40])


@pytest.mark.gpu
def test_recognizer_with_more_than_1024_patches():
    cfg = dataclasses.replace(SMALL, image_size=528)
    assert cfg.tokens == 1090
    ref = model(cfg)
    x, xin = image(cfg, 2, "cuda")
    toks, _ = model(cfg).cuda().prepare().generate(xin, max_len=10)
    check_tokens(ref, x, toks)


@pytest.mark.parametrize("dev", DEVICES)
def test_recognizer_with_4_bit_weights(dev):
    """The tokens are those of the PyTorch model whose decoder weights are the 4-bit ones."""
    ref = model(SMALL)
    with torch.no_grad():
        for l in ref.dec:
            for lin in (l.qkv, l.proj, l.xq, l.xproj, l.fc1, l.fc2):
                lin.weight.copy_(Q.quantize_int4(lin.weight, 64).dequantize())
        ref.lm_head.weight.copy_(Q.quantize_int4(ref.lm_head.weight, 64).dequantize())
    x, xin = image(SMALL, 3, dev)
    m = model(SMALL).to(dev).prepare(int4_group=64)
    assert isinstance(m._pk["dec"][0]["qkv"][0], Q.Int4Weight)
    toks, _ = m.generate(xin, max_len=10)
    check_tokens(ref, x, toks)
    m = m.to(dev)                               # packed weights are dropped; the choice stays
    assert m._pk is None
    again, _ = m.generate(xin, max_len=10)
    assert torch.equal(again, toks) and isinstance(m._pk["lm"][0], Q.Int4Weight)
    assert not isinstance(m.prepare(int4_group=0)._pk["lm"][0], Q.Int4Weight)


def test_rules_give_what_the_entries_take():
    """Launch shapes over the whole range of sizes lie within the kernels' own checks."""
    if not _loader.kernels_available():
        pytest.skip("the kernel library is not built")
    rules, g = _loader.bind(), random.Random(0)
    log = lambda hi: int(math.exp(g.uniform(0, math.log(hi))))  # noqa: E731
    for _ in range(4000):
        m, n, k = log(1 << 20), log(1 << 26), log(1 << 23)
        tiles, nw, kw, kz = rules.rule_shape(m, n, k)
        wide = 1 if m <= 16 else 2
        assert tiles in (1, 2 * wide) and nw >= 1 and kw >= 1 and nw * kw <= 8 and nw * kw * tiles * wide <= 64 and 1 <= kz <= 64
        assert kw * kz <= max(1, -(-k // 128)) * 4
        share, least = rules.rule_deal(log(1 << 23), log(48), log(1 << 30), g.choice((64, 128)))
        assert (share, least) == (0, 0) or (0 < share <= 1 << 20 and least >= 1)
        b, v = log(1 << 22), log(1 << 29)
        pieces = rules.rule_pieces(b, v)
        assert 1 <= pieces <= 64 and (pieces == 1 or b <= 65535)


@pytest.mark.parametrize("dev", DEVICES)
def test_a_refused_group_changes_nothing(dev):
    """Sizes of groups that no layer has: the weights packed before, or none, and the earlier choice stand."""
    _, xin = image(SMALL, 2, dev)
    m = model(SMALL).to(dev)
    for bad in (48, 256):
        with pytest.raises(ValueError):
            m.prepare(int4_group=bad)
    toks, _ = m.generate(xin, max_len=4)
    assert m.int4_group == 0 and not isinstance(m._pk["lm"][0], Q.Int4Weight)
    m.prepare(int4_group=32)
    four, _ = m.generate(xin, max_len=4)
    with pytest.raises(ValueError):
        m.prepare(int4_group=48)
    assert m.int4_group == 32 and torch.equal(m.generate(xin, max_len=4)[0], four)
    m = m.to(dev)                               # packed weights are dropped; the choice stays
    assert torch.equal(m.generate(xin, max_len=4)[0], four) and m._pk["lm"][0].group == 32


@pytest.mark.gpu
def test_without_a_graph_nothing_is_replayed():
    """Eager steps after captured ones, and the other way round: each call does as it is told, with the same tokens."""
    _, xin = image(SMALL, 3, "cuda")
    for first in (True, False):
        m, want = model(SMALL).cuda().prepare(), None
        replays = lambda: sum(g.replays for g in m._graphs.values())  # noqa: E731
        for use_graph in (first, not first, first):
            before = replays()
            toks, conf = m.generate(xin, use_graph=use_graph, eos_check_every=0)
            assert replays() - before == (SMALL.max_len if use_graph else 0)
            want = want or (toks, conf)
            assert torch.equal(toks, want[0]) and torch.equal(conf, want[1])


@pytest.mark.gpu
def test_recognizer_over_its_whole_length():
    """Sequences that cannot end: every token up to the last position, across page borders and beyond 1024, is compared with the
    PyTorch model; the captured step and the eager one give the same."""
    cfg = dataclasses.replace(SMALL, max_len=1100)
    models = [model(cfg, seed=1) for _ in range(2)]
    for m in models:
        with torch.no_grad():
            m.lm_head.weight[cfg.eos] = 0.0                    # a logit of 0 never is the largest of 300
    x, xin = image(cfg, 2, "cuda")
    m = models[1].cuda().prepare()
    toks, conf = m.generate(xin)
    assert toks.shape == (2, 1100) and not bool((toks == cfg.eos).any()) and m.last_decode_steps == 1100
    near = check_tokens(models[0], x, toks)
    for part in (slice(0, 64), slice(64, 1024), slice(1024, 1100)):
        assert near[:, part].float().mean().item() > 0.9, part
    before = sum(g.replays for g in m._graphs.values())
    eager, econf = m.generate(xin, use_graph=False)
    assert sum(g.replays for g in m._graphs.values()) == before
    assert torch.equal(eager, toks) and torch.equal(econf, conf)
