"""Cases of the operators of a small-batch decode step: keys and values appended to a paged cache (with the position
rotation on the way), attention of the new tokens over that cache, linear layers with 4-bit weights, and the
verification of drafted tokens.

``own`` False: the operators in plain torch operations, 32 bits (64 where borders decide).  ``own`` True: the calls a
user makes of ``distributed_llms_amd.ops``.  ``exact`` says what either should return, in 64 bits."""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of the line recognizer's decoder (16 heads of 64, learned positions: nothing to rotate) for
        # its smallest batch bucket.
        {"name": "append step", "op": "append", "batch": 16, "tokens": 16, "ragged": False, "q_heads": 0, "kv_heads": 16,
         "dim": 64, "rot": 0, "interleaved": False, "page": 16, "past": 128, "dtype": "bf16"},
        # Four drafted tokens and the last sampled one of 32 sequences, grouped heads, queries rotated in the same call.
        {"name": "append drafted", "op": "append", "batch": 32, "tokens": 160, "ragged": False, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "interleaved": False, "page": 64, "past": 4000, "dtype": "fp16"},
        # Prompts of many lengths packed one behind the other (some continue a cached part), half of the dimensions
        # rotated in neighbouring pairs: the largest call.
        {"name": "append prompts", "op": "append", "batch": 48, "tokens": 16384, "ragged": True, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 64, "interleaved": True, "page": 32, "past": 700, "dtype": "bf16"},
        # Self-attention of one decode step of the line recognizer: short lines, a page of 16 tokens.
        {"name": "attend lines", "op": "attend", "batch": 16, "new": 1, "q_heads": 16, "kv_heads": 16, "dim": 64, "page": 16,
         "longest": 128, "ragged": True, "causal": True, "lse": False, "dtype": "bf16"},
        # Cross-attention of a decode step: 577 encoder tokens of 64 crops held in pages.
        {"name": "attend memory", "op": "attend", "batch": 64, "new": 1, "q_heads": 16, "kv_heads": 16, "dim": 64, "page": 32,
         "longest": 577, "ragged": False, "causal": False, "lse": False, "dtype": "bf16"},
        # Drafted tokens over caches of very different lengths, grouped heads.
        {"name": "attend drafted", "op": "attend", "batch": 12, "new": 5, "q_heads": 32, "kv_heads": 4, "dim": 128, "page": 48,
         "longest": 8009, "ragged": True, "causal": True, "lse": True, "dtype": "fp16"},
        # One user with one long document: the whole card works on a single sequence.
        {"name": "attend long", "op": "attend", "batch": 1, "new": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "longest": 100003, "ragged": False, "causal": True, "lse": False, "dtype": "bf16"},
        # Drafts of four tokens for one sequence, the line recognizer's vocabulary.
        {"name": "verify one", "op": "verify", "batch": 1, "drafted": 4, "vocab": 50265, "proposal": True, "dtype": "fp32"},
        # A full batch of drafts.
        {"name": "verify batch", "op": "verify", "batch": 192, "drafted": 7, "vocab": 50265, "proposal": True, "dtype": "fp32"},
        # First feed-forward layer of the line recognizer's decoder for one sequence.
        {"name": "int4 layer", "op": "int4", "rows": 1, "n": 4096, "k": 1024, "group": 64, "zero": False, "act": "gelu",
         "res": False, "dtype": "bf16"},
        # Its vocabulary projection for five tokens (four drafted ones and the last sampled one): an odd number of outputs.
        {"name": "int4 vocabulary", "op": "int4", "rows": 5, "n": 50265, "k": 1024, "group": 128, "zero": True, "act": "none",
         "res": False, "dtype": "bf16"},
        # A wide layer for a small batch, with the residual added.
        {"name": "int4 wide", "op": "int4", "rows": 24, "n": 8192, "k": 28672, "group": 128, "zero": True, "act": "none",
         "res": True, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "verify", "int4"])
    if op == "append":
        dim = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8, 12, 16])
        rot = rng.choice([0, dim // 2, dim])
        batch = _log(rng, 1, 64)
        ragged = rng.random() < 0.5
        tokens = _log(rng, max(batch, 2), 8000) if ragged else batch * _log(rng, 1, 16)
        return {"op": op, "batch": batch, "tokens": tokens, "ragged": ragged,
                "q_heads": kv * rng.choice([1, 2, 4]) if rot else 0, "kv_heads": kv, "dim": dim, "rot": rot,
                "interleaved": rng.random() < 0.5, "page": 16 * rng.choice([1, 2, 3, 4, 8]), "past": _log(rng, 1, 4000),
                "dtype": rng.choice(["bf16", "fp16"])}
    if op == "attend":
        causal = rng.random() < 0.75
        kv, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 4, 8])
        batch = _log(rng, 1, 64)
        longest = max(16, _log(rng, 16, min(65536, 800000 // (batch * kv))))
        return {"op": op, "batch": batch, "new": rng.choice([1, 1, 2, 3, 5, 8]), "q_heads": kv * group, "kv_heads": kv,
                "dim": rng.choice([64, 128]), "page": 16 * rng.choice([1, 2, 3, 4, 8]), "longest": longest,
                "ragged": rng.random() < 0.7, "causal": causal, "lse": rng.random() < 0.4, "dtype": rng.choice(["bf16", "fp16"])}
    if op == "verify":
        return {"op": op, "batch": _log(rng, 1, 128), "drafted": rng.randint(1, 7), "vocab": _log(rng, 200, 80000),
                "proposal": rng.random() < 0.7, "dtype": rng.choice(["fp32", "fp32", "bf16"])}
    group = rng.choice([32, 64, 128])
    return {"op": op, "rows": _log(rng, 1, 48), "n": _log(rng, 200, 20000), "k": group * _log(rng, 2, 8192 // group),
            "group": group, "zero": rng.random() < 0.5, "act": rng.choice(["none", "none", "gelu", "relu"]),
            "res": rng.random() < 0.3, "dtype": rng.choice(["bf16", "fp16"])}


# Lengths belong to the case, not to the seed: the work of a case is one number.
def _append_lens(c):
    r = random.Random(c["batch"] * 7919 + c["tokens"] * 31 + c["past"])
    past = [r.randint(0, c["past"]) for _ in range(c["batch"])]
    if not c["ragged"]:
        return past, [c["tokens"] // c["batch"]] * c["batch"], 0
    behind = c["tokens"] // 64                         # rows behind the last sequence: padding of the token batch
    cuts = sorted(r.randint(0, c["tokens"] - behind) for _ in range(c["batch"] - 1))
    ends = [0] + cuts + [c["tokens"] - behind]
    return past, [b - a for a, b in zip(ends, ends[1:])], behind


def _attend_lens(c):
    r = random.Random(c["batch"] * 7919 + c["longest"] * 31 + c["page"])
    top = c["longest"]
    lens = [top] * c["batch"] if not c["ragged"] else [_log(r, 1, top) if r.random() < 0.5 else r.randint(1, top) for _ in range(c["batch"])]
    lens[-1] = top
    if c["causal"]:
        return [max(0, n - c["new"]) for n in lens]     # tokens kept before the step; the new ones follow them
    if c["ragged"] and c["batch"] > 1:
        lens[0] = 0                                    # a sequence without any memory
    return lens


# ------------------------------------------------------------------------------------------------ inputs
def _table(needed, page, width, gen, dev):
    """Random distinct pages for every sequence; entries behind a sequence's last page are -1."""
    counts = [-(-n // page) for n in needed]
    total = sum(counts) + 3
    perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    flat = torch.arange(width, device=dev)[None, :]
    cnt = torch.tensor(counts, device=dev)
    start = cnt.cumsum(0) - cnt
    at = (start[:, None] + flat).clamp(max=total - 1)
    return torch.where(flat < cnt[:, None], perm[at], torch.full_like(perm[at], -1)).contiguous(), total


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    c, dt = dict(case), TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=None):
        x = torch.empty(shape, dtype=dt if dtype is None else dtype, device=dev).normal_(generator=g)
        return x if scale == 1.0 else x.mul_(scale)

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = {"case": c}
    if c["op"] == "append":
        past, new, _ = _append_lens(c)
        need = [p + n for p, n in zip(past, new)]
        width = max(1, -(-max(need) // c["page"]))
        s["table"], pages = _table(need, c["page"], width, g, dev)
        s["k_pages"], s["v_pages"] = (normal(pages, c["page"], c["kv_heads"], c["dim"]) for _ in range(2))
        # queries, keys and values are slices of one fused projection
        T, hq, hkv, d = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"]
        qkv = normal(T, (hq + 2 * hkv), d)
        s["q"] = qkv[:, :hq] if hq else None
        s["k"], s["v"] = qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
        s["lens"] = i32(past)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["starts"] = i32(starts) if c["ragged"] else None
        s["cos"] = s["sin"] = None
        if c["rot"]:
            half = c["rot"] // 2
            freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
            ang = torch.arange(width * c["page"], dtype=torch.float64, device=dev)[:, None] * freq
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    elif c["op"] == "attend":
        lens = _attend_lens(c)
        need = [n + (c["new"] if c["causal"] else 0) for n in lens]
        s["table"], pages = _table(need, c["page"], max(1, -(-max(need) // c["page"])), g, dev)
        s["k_pages"], s["v_pages"] = (normal(pages, c["page"], c["kv_heads"], c["dim"]) for _ in range(2))
        s["q"] = normal(c["batch"], c["new"], c["q_heads"], c["dim"], scale=2.0)
        s["lens"] = i32(lens)
    elif c["op"] == "verify":
        B, n, V = c["batch"], c["drafted"], c["vocab"]
        logits = normal(B, n + 1, V, scale=2.5, dtype=torch.float32)
        s["target"] = torch.softmax(logits, -1).to(dt)
        prop = logits[:, :n] + normal(B, n, V, scale=0.4, dtype=torch.float32)
        s["proposal"] = torch.softmax(prop, -1).to(dt) if c["proposal"] else None
        e = torch.empty((B, n, V), device=dev).exponential_(generator=g)
        s["draft"] = (prop - e.log()).argmax(-1).to(torch.int32)      # one token drawn from each row
        s["u"] = torch.rand((B, n + 1), generator=g, device=dev)
        r = random.Random(B * 31 + n)
        s["counts"] = i32([n if r.random() < 0.8 else r.randint(0, n) for _ in range(B)])
    else:
        N, K, G = c["n"], c["k"], c["group"]
        s["packed"] = torch.randint(0, 256, (N, K // 2), generator=g, device=dev, dtype=torch.uint8)   # low nibble first
        s["scale"] = ((torch.rand((N, K // G), generator=g, device=dev) + 0.5) * (0.25 / math.sqrt(K))).to(dt)
        s["zero"] = torch.randint(4, 12, (N, K // G), generator=g, device=dev, dtype=torch.uint8) if c["zero"] else None
        s["x"] = normal(c["rows"], K)
        s["bias"] = torch.empty((N,), device=dev).normal_(generator=g) * 0.1
        s["res"] = normal(c["rows"], N) if c["res"] else None
        if own:
            # what a program keeps of a layer: the weights in the kernels' order, once
            from distributed_llms_amd.ops.int4 import pack_int4

            s["weight"] = pack_int4(s["packed"], s["scale"], s["zero"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _append, "attend": _attend, "verify": _verify, "int4": _int4}[op](s)
    c = s["case"]
    if op == "append":
        from distributed_llms_amd.ops.paged import paged_append

        q = paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], q=s["q"], cos=s["cos"], sin=s["sin"],
                         starts=s["starts"], interleaved=c["interleaved"])
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "q": q}
    if op == "attend":
        from distributed_llms_amd.ops.paged import paged_attention

        r = paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], causal=c["causal"], return_lse=c["lse"])
        return {"o": r[0], "lse": r[1]} if c["lse"] else {"o": r}
    if op == "verify":
        from distributed_llms_amd.ops.draft import verify_draft

        tokens, accepted = verify_draft(s["draft"], s["target"], s["u"], proposal=s["proposal"], counts=s["counts"])
        return {"tokens": tokens, "accepted": accepted}
    from distributed_llms_amd.ops.int4 import linear_int4

    return linear_int4(s["x"], s["weight"], s["bias"], act=c["act"], res=s["res"])


def _rotate(x, cos, sin, rot, interleaved):
    """x [T, H, D] float; the first ``rot`` dimensions turn by the angles of cos / sin [T, rot / 2]."""
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
    cos, sin = cos[:, None], sin[:, None]
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _append(s):
    c, table, page = s["case"], s["table"], s["case"]["page"]
    T = c["tokens"]
    t = torch.arange(T, device=table.device)
    if s["starts"] is None:
        seq = t // (T // c["batch"])
        first = seq * (T // c["batch"])
        last = None
    else:
        last = s["starts"][-1].long()
        t = torch.minimum(t, last - 1)                 # rows behind the last sequence write its last token once more
        seq = (s["starts"][1:].long()[None, :] <= t[:, None]).sum(1)
        first = s["starts"].long()[seq]
    pos = s["lens"].long()[seq] + t - first
    where = table.long()[seq, pos // page] * page + pos % page
    k, v, q = s["k"], s["v"], s["q"]
    if last is not None:
        k, v = k[t], v[t]
    if c["rot"]:
        cos, sin = s["cos"][pos], s["sin"][pos]
        k = _rotate(k.float(), cos, sin, c["rot"], c["interleaved"])
        q = _rotate(q.float(), cos, sin, c["rot"], c["interleaved"])
        if last is not None:
            q = q * (torch.arange(T, device=q.device) < last)[:, None, None]   # no sequence: no query
        q = q.to(s["q"].dtype)
    s["k_pages"].view(-1, *k.shape[1:])[where] = k.to(s["k_pages"].dtype)
    s["v_pages"].view(-1, *v.shape[1:])[where] = v
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "q": q}


def _attend(s):
    c, q = s["case"], s["q"]
    B, n, hq, d = q.shape
    hkv = c["kv_heads"]
    idx = s["table"].long().clamp(min=0)
    L = idx.shape[1] * c["page"]
    k = s["k_pages"][idx].reshape(B, L, hkv, d).permute(0, 2, 1, 3).float()
    v = s["v_pages"][idx].reshape(B, L, hkv, d).permute(0, 2, 1, 3).float()
    qf = q.float().view(B, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, d)
    x = (qf @ k.transpose(-1, -2)) / math.sqrt(d)      # [B, hkv, n * group, L]
    seen = s["lens"].long()[:, None] + (torch.arange(1, n + 1, device=q.device) if c["causal"] else torch.zeros(n, device=q.device, dtype=torch.long))
    mask = torch.arange(L, device=q.device) < seen[..., None]                   # [B, n, L]
    mask = mask[:, None, :, None].expand(B, hkv, n, hq // hkv, L).reshape(x.shape)
    x = x.masked_fill(~mask, float("-inf"))
    top = x.amax(-1, keepdim=True)
    e = torch.where(mask, (x - top).exp(), torch.zeros((), device=q.device))    # a row without keys: all zeros
    total = e.sum(-1, keepdim=True)
    o = (e @ v) / total.clamp(min=1e-30)
    back = lambda y: y.reshape(B, hkv, n, hq // hkv, -1).permute(0, 2, 1, 3, 4).reshape(B, n, hq, -1)  # noqa: E731
    o = back(o).to(q.dtype)
    return {"o": o, "lse": back(top + total.log())[..., 0].contiguous()} if c["lse"] else {"o": o}


def _verify(s):
    c, draft = s["case"], s["draft"].long()
    B, n = draft.shape
    i = torch.arange(n, device=draft.device)
    p = s["target"][:, :n].gather(2, draft[..., None])[..., 0].double()
    q = s["proposal"].gather(2, draft[..., None])[..., 0].double() if s["proposal"] is not None else torch.ones_like(p)
    ok = (s["u"][:, :n].double() * q < p) & (i < s["counts"][:, None])
    taken = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device=draft.device)
    row = s["target"][b, taken].double()
    at = taken.clamp(max=n - 1)
    rest = (taken < s["counts"]).double()[:, None]
    if s["proposal"] is not None:
        less = s["proposal"][b, at].double()
    else:
        less = (torch.arange(c["vocab"], device=draft.device) == draft[b, at][:, None]).double()   # all of it on the drafted token
    left = (row - less * rest).clamp(min=0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, row)
    cdf = left.cumsum(1)
    new = (cdf <= s["u"][:, n:].double() * cdf[:, -1:]).sum(1).clamp(max=c["vocab"] - 1)
    j = torch.arange(n + 1, device=draft.device)
    full = torch.cat((draft, draft[:, -1:]), 1)
    tokens = torch.where(j < taken[:, None], full, torch.where(j == taken[:, None], new[:, None], torch.full_like(full, -1)))
    return {"tokens": tokens.to(torch.int32), "accepted": taken.to(torch.int32)}


def _int4(s):
    c, w = s["case"], s["packed"]
    q = torch.stack((w & 15, w >> 4), -1).view(c["n"], c["k"] // c["group"], c["group"]).float()
    z = s["zero"].float() if s["zero"] is not None else torch.full_like(q[..., 0], 8.0)
    wf = ((q - z[..., None]) * s["scale"].float()[..., None]).view(c["n"], c["k"])
    y = s["x"].float() @ wf.t() + s["bias"]
    if s["res"] is not None:
        y = y + s["res"].float()
    if c["act"] == "relu":
        y = y * (y > 0)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * 0.5 ** 0.5))
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------------------------------------ floors and truth
def work(c):
    e = SIZE[c["dtype"]]
    if c["op"] == "append":
        past, new, _ = _append_lens(c)
        T = sum(new)
        kv = 2 * T * c["kv_heads"] * c["dim"] * e * 2
        q = (T + c["tokens"]) * c["q_heads"] * c["dim"] * e
        angles = len({p + i for p, n in zip(past, new) for i in range(n)}) * c["rot"] * 4
        return {"bytes": kv + q + angles, "flops": 3 * T * (c["q_heads"] + c["kv_heads"]) * c["rot"]}
    if c["op"] == "attend":
        lens = _attend_lens(c)
        more = c["new"] if c["causal"] else 0
        keys = sum(n + more for n in lens)
        kv = 2 * keys * c["kv_heads"] * c["dim"] * e
        q = 2 * c["batch"] * c["new"] * c["q_heads"] * c["dim"] * e
        seen = sum((n + (i + 1 if c["causal"] else 0)) for n in lens for i in range(c["new"]))
        return {"bytes": kv + q, "flops": 4 * seen * c["q_heads"] * c["dim"]}
    if c["op"] == "verify":
        # the drafted tokens' probabilities, then for each sequence one row of the target and one of the proposal
        rows = c["batch"] * (2 if c["proposal"] else 1)
        return {"bytes": rows * c["vocab"] * e + c["batch"] * c["drafted"] * 2 * e, "flops": 2 * rows * c["vocab"]}
    groups = c["n"] * c["k"] // c["group"]
    return {"bytes": c["n"] * c["k"] // 2 + groups * (e + (1 if c["zero"] else 0)) + c["rows"] * (c["k"] + c["n"] * (2 if c["res"] else 1)) * e + 4 * c["n"],
            "flops": 2 * c["rows"] * c["n"] * c["k"]}


def exact(case, seed):
    """The outputs from the operators' definitions, sequence by sequence, in 64 bits."""
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "append":
        past, new, _ = _append_lens(c)
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        qo = torch.zeros(s["q"].shape, dtype=torch.float64, device=kp.device) if s["q"] is not None else None
        at = 0
        for b, (p, n) in enumerate(zip(past, new)):
            if n == 0:
                continue
            pos = torch.arange(p, p + n, device=kp.device)
            page, slot = s["table"][b, pos // c["page"]].long(), pos % c["page"]
            vp[page, slot] = s["v"][at : at + n].double()
            k = s["k"][at : at + n].double()
            if c["rot"]:
                w = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
                k, q = _turn(k, w, c), _turn(s["q"][at : at + n].double(), w, c)
                qo[at : at + n] = q
            kp[page, slot] = k
            at += n
        return {"k_pages": kp, "v_pages": vp, "q": qo}
    if c["op"] == "attend":
        q = s["q"].double()
        B, n, hq, d = q.shape
        group = hq // c["kv_heads"]
        o, lse = torch.zeros_like(q), torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
        for b, kept in enumerate(_attend_lens(c)):
            for i in range(n):
                seen = kept + i + 1 if c["causal"] else kept
                if seen == 0:
                    continue
                pos = torch.arange(seen, device=q.device)
                page, slot = s["table"][b, pos // c["page"]].long(), pos % c["page"]
                k, v = s["k_pages"][page, slot].double(), s["v_pages"][page, slot].double()    # [seen, hkv, d]
                qg = q[b, i].view(-1, group, d)
                x = torch.bmm(qg, k.permute(1, 2, 0).contiguous()) * d ** -0.5
                lse[b, i] = torch.logsumexp(x, -1).reshape(-1)
                o[b, i] = torch.bmm(torch.softmax(x, -1), v.transpose(0, 1).contiguous()).reshape(hq, d)
        return {"o": o, "lse": lse} if c["lse"] else {"o": o}
    if c["op"] == "int4":
        lo, hi = s["packed"].long() % 16, s["packed"].long() // 16
        at = torch.arange(c["k"], device=lo.device)
        q = torch.where(at % 2 == 0, lo.repeat_interleave(2, 1), hi.repeat_interleave(2, 1)).double()
        zero = 8.0 if s["zero"] is None else s["zero"].double().repeat_interleave(c["group"], 1)
        w = (q - zero) * s["scale"].double().repeat_interleave(c["group"], 1)
        y = torch.mm(s["x"].double(), w.t().contiguous()) + s["bias"].double()
        y = y if s["res"] is None else y + s["res"].double()
        return y.clamp(min=0) if c["act"] == "relu" else y * 0.5 * torch.erfc(-y / math.sqrt(2)) if c["act"] == "gelu" else y
    return None                                         # whole numbers: compared as they are


def _turn(x, w, c):
    """x [T, H, D] in 64 bits; pairs of its first ``rot`` dimensions as complex numbers, multiplied by w [T, 1, rot / 2]."""
    r = c["rot"]
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * w
        y = torch.view_as_real(z).reshape(*x.shape[:-1], r)
    else:
        z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2 : r].contiguous()) * w
        y = torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., r:]), -1)
