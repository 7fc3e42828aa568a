"""Attention over a paged K/V cache for several sequences, as cases that can be timed and checked.

The cache is a pair of tensors [pages, Hk, page, D]; sequence b's position p is row p % page of page
table[b, p // page]. Four operators fill and read it:

  append   head norms, rotation and storing of new tokens' keys and values (kernels.kv_append)
  prompt   causal attention of packed prompts (kernels.attn_prompt)
  batch    one token per sequence (kernels.attn_batch)
  shared   one token per sequence, after a prefix that all sequences share (kernels.attn_shared)

`run` computes them in plain torch in 32 bits, or, with `own`, through the package's entry points;
`exact` restates them in 64 bits. Head shapes are those of the models that the package serves
(32 query and 4 key/value heads of 128, 64 and 8 of 64, 16 and 2 of 256) and generic ones.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    q3 = dict(hq=32, hk=4, d=128, page=64, dtype="bf16", hole=False)  # Qwen3-30B-A3B's heads
    oss = dict(hq=64, hk=8, d=64, dtype="f16", hole=False)  # gpt-oss-20b's heads
    return [
        # the new tokens of eight decoding sequences: the smallest call of a serving step
        dict(name="append_step8", kind="append", B=8, lo=1, hi=1, ctx=4000, rot=128, norm=True, inter=False, pick=1, **q3),
        # five prompts admitted together
        dict(name="append_prompts", kind="append", B=5, lo=300, hi=2500, ctx=0, rot=128, norm=True, inter=False, pick=2, **q3),
        # wide heads rotated in part, pairs interleaved, prompts that continue cached turns
        dict(name="append_partial", kind="append", B=6, lo=200, hi=3000, ctx=5000, rot=64, norm=True, inter=True, pick=3,
             hq=16, hk=2, d=256, page=16, dtype="f16", hole=False),
        # a short question: latency counts
        dict(name="prompt_61", kind="prompt", B=1, lo=61, hi=61, ctx=0, pick=4, **q3),
        # seven prompts of different lengths in one pack
        dict(name="prompt_pack7", kind="prompt", B=7, lo=100, hi=4000, ctx=0, pick=5, **q3),
        # one long document
        dict(name="prompt_16k", kind="prompt", B=1, lo=16384, hi=16384, ctx=0, pick=6, **q3),
        # the next chunks of two long prompts whose beginnings are cached
        dict(name="prompt_chunk", kind="prompt", B=2, lo=509, hi=509, ctx=24000, pick=7, page=32, **oss),
        # a decode step of one sequence: latency counts
        dict(name="batch_1", kind="batch", B=1, lo=1009, hi=1009, pick=8, **q3),
        # a decode step of 32 sequences of very different lengths
        dict(name="batch_32", kind="batch", B=32, lo=200, hi=16000, pick=9, **q3),
        # two sequences with very long contexts
        dict(name="batch_long", kind="batch", B=2, lo=100000, hi=130000, pick=10, page=128, **oss),
        # eight samples of one answer
        dict(name="shared_8", kind="shared", B=8, lo=1, hi=200, prefix=1531, pick=11, **q3),
        # 64 requests behind one long system prompt
        dict(name="shared_64", kind="shared", B=64, lo=50, hi=900, prefix=16000, pick=12, **q3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 4, 128), (32, 8, 128), (64, 8, 64), (16, 2, 256), (8, 8, 128), (16, 16, 64), (28, 4, 128), (40, 8, 128),
          (12, 2, 64), (32, 2, 128)]


def draw(rng):
    kind = rng.choice(["append", "prompt", "prompt", "batch", "batch", "shared"])
    hq, hk, d = rng.choice(_HEADS)
    c = dict(kind=kind, hq=hq, hk=hk, d=d, page=rng.choice([16, 32, 64, 128, 256]), dtype=rng.choice(["bf16", "bf16", "f16"]),
             pick=rng.randrange(1 << 30), hole=rng.random() < 0.25)
    wide = hq * d / 4096  # against the listed cases' heads
    if kind == "append":
        c["B"] = _log_int(rng, 1, 24)
        c["hole"] &= c["B"] > 1
        most = max(1, int(9000 / wide) // c["B"])
        a, b = sorted((_log_int(rng, 1, most), _log_int(rng, 1, most)))
        return dict(c, lo=a, hi=b, ctx=rng.choice([0, 300, 6000]), rot=rng.choice([d, d, d // 2, d // 4]), norm=rng.random() < 0.6,
                    inter=rng.random() < 0.4)
    if kind == "prompt":
        c["B"] = _log_int(rng, 1, 12)
        c["hole"] &= c["B"] > 1
        ctx = rng.choice([0, 0, 500, 9000])
        most = int(9000 / wide / c["B"] ** 0.5) if ctx == 0 else int(2500 / wide / c["B"])
        a, b = sorted((_log_int(rng, 1, most), _log_int(rng, 1, most)))
        return dict(c, lo=a, hi=b, ctx=ctx)
    c["B"] = _log_int(rng, 1, 64)
    c["hole"] &= c["B"] > 1
    per = hk * d / 512
    if kind == "batch":
        most = max(64, min(100000, int(150000 / per) // c["B"]))
        a, b = sorted((_log_int(rng, 1, most), _log_int(rng, 1, most)))
        return dict(c, lo=a, hi=b)
    a, b = sorted((_log_int(rng, 1, 900 / per), _log_int(rng, 1, 900 / per)))
    return dict(c, lo=a, hi=b, prefix=_log_int(rng, 10, 14000 / per))


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """(new tokens, cached positions before them) of each sequence; batch and shared: positions and zeros."""
    rng = random.Random(case["pick"])
    n = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["B"])]
    ctx = [rng.randint(case.get("ctx", 0) // 2, case.get("ctx", 0)) for _ in n]
    if case["hole"]:  # a slot of the batch that holds no sequence
        n[0] = ctx[0] = 0
    return n, ctx


def _randn(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _paged(case, gen, lens, extra):
    """Page tables of `lens` positions each over randomly ordered pages, and the filled cache ("extra" pages more)."""
    page, dt = case["page"], DT[case["dtype"]]
    need = [-(-n // page) for n in lens]
    P = sum(need) + extra
    order = torch.randperm(P, generator=gen, device=DEV).to(torch.int32)
    tables, at = [], 0
    for n in need:
        tables.append(order[at : at + n])
        at += n
    table = torch.zeros((len(lens), max(1, max(need))), dtype=torch.int32, device=DEV)
    for b, t in enumerate(tables):
        table[b, : t.numel()] = t
    shape = (P, case["hk"], page, case["d"])
    return table, _randn(gen, shape, dt), _randn(gen, shape, dt)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 9973 + 17)
    n, ctx = _lengths(case)
    hq, hk, d, dt, kind = case["hq"], case["hk"], case["d"], DT[case["dtype"]], case["kind"]
    total = [a + b for a, b in zip(n, ctx)]
    s = dict(case, scale=d**-0.5, new=n, total=total)
    if kind == "shared":
        table, s["kc"], s["vc"] = _paged(case, gen, total + [case["prefix"]], 3)
        s["prefix_table"] = table[-1, : -(-case["prefix"] // case["page"])].contiguous()
        s["prefix_len"] = _ints([case["prefix"]])
        s["table"] = table[:-1, : max(1, -(-max(total) // case["page"]))].contiguous()
    else:
        s["table"], s["kc"], s["vc"] = _paged(case, gen, total, 3)
    s["kv_len"] = _ints(total)
    if kind in ("append", "prompt"):
        cu = [0]
        for a in n:
            cu.append(cu[-1] + a)
        s["cu"] = _ints(cu)
        T = cu[-1]
    else:
        T = case["B"]
    if kind == "append":
        qkv = _randn(gen, (T, hq + 2 * hk, d), dt)  # the fused projection's output
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq : hq + hk], qkv[:, hq + hk :]
        s["qn"] = _randn(gen, (d,), dt, 0.1) + 1 if case["norm"] else None
        s["kn"] = _randn(gen, (d,), dt, 0.1) + 1 if case["norm"] else None
        rot = case["rot"]
        inv = 1.0 / (1e6 ** (torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot))
        ang = torch.arange(max(total) + 1, device=DEV, dtype=torch.float64)[:, None] * inv[None]
        ang = ang.repeat_interleave(2, 1) if case["inter"] else torch.cat([ang, ang], 1)
        s["cos"], s["sin"] = ang.cos().to(dt), ang.sin().to(dt)
    else:
        s["q"] = _randn(gen, (T, hq, d), dt)
    return s


# ------------------------------------------------------------------ one pass
def _places(s):
    """Page and row of every new token, from the lengths on the device."""
    cu, kv, page = s["cu"].long(), s["kv_len"].long(), s["page"]
    tok = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(cu[1:], tok, right=True)
    pos = kv[b] - (cu[b + 1] - tok)
    return pos, s["table"][b, pos // page].long(), pos % page


def _plain_append(s):
    pos, pg, row = _places(s)
    rot = s["rot"]
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]

    def head(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        r = x[..., :rot]
        if s["inter"]:
            turned = torch.stack([-r[..., 1::2], r[..., 0::2]], -1).flatten(-2)
        else:
            turned = torch.cat([-r[..., rot // 2 :], r[..., : rot // 2]], -1)
        return torch.cat([r * cos + turned * sin, x[..., rot:]], -1).to(s["q"].dtype)

    q = head(s["q"], s["qn"])
    s["kc"][pg, :, row] = head(s["k"], s["kn"])
    s["vc"][pg, :, row] = s["v"]
    return dict(q=q, kc=s["kc"], vc=s["vc"])


def _gather(cache, pages, length):
    """Positions [0, length) of the listed pages: float [Hk, length, D]."""
    rows = cache[pages.long()].float()  # [n, Hk, page, D]
    return rows.transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :length]


def _softmax_rows(q, k, v, scale, first):
    """q [Hq, n, D] at positions first .. first + n - 1 over k, v [Hk, len, D]: [n, Hq, D], in blocks of rows."""
    hq, n, d = q.shape
    hk, length = k.shape[:2]
    g = hq // hk
    out = torch.zeros((n, hq, d), device=DEV)
    if length == 0:
        return out
    cols = torch.arange(length, device=DEV)
    block = max(1, (1 << 28) // (g * length))
    for h in range(hk):
        kt = k[h].t().contiguous()
        for i in range(0, n, block):
            m = min(block, n - i)
            sc = (q[h * g : (h + 1) * g, i : i + m].reshape(g * m, d) @ kt) * scale
            sc = sc.view(g, m, length).masked_fill_(cols > (first + i + torch.arange(m, device=DEV))[:, None], -math.inf)
            sc = (sc - sc.amax(-1, keepdim=True)).exp_()
            o = (sc.view(g * m, length) @ v[h]) / sc.sum(-1).view(g * m, 1)
            out[i : i + m, h * g : (h + 1) * g] = o.view(g, m, d).transpose(0, 1)
    return out


def _plain_attend(s):
    q, page = s["q"], s["page"]
    head, t = 0, 0
    if s["kind"] == "shared":
        head = s["prefix"]
        pk, pv = _gather(s["kc"], s["prefix_table"], head), _gather(s["vc"], s["prefix_table"], head)
    out = torch.zeros_like(q)
    for b, length in enumerate(s["total"]):
        n = s["new"][b] if s["kind"] == "prompt" else 1
        pages = s["table"][b, : -(-length // page)]
        k, v = _gather(s["kc"], pages, length), _gather(s["vc"], pages, length)
        if head:
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        rows = q[t : t + n].float().transpose(0, 1)
        out[t : t + n] = _softmax_rows(rows, k, v, s["scale"], head + length - n).to(q.dtype)
        t += n
    return out


def _own(s):
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wisp-runtime_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from wisp import kernels

    kind = s["kind"]
    if kind == "append":
        q = kernels.kv_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["cu"], s["kv_len"], s["table"], s["kc"], s["vc"],
                              q_norm_w=s["qn"], k_norm_w=s["kn"], eps=EPS, interleaved=s["inter"])
        return dict(q=q, kc=s["kc"], vc=s["vc"])
    if kind == "prompt":
        return kernels.attn_prompt(s["q"], s["kc"], s["vc"], s["cu"], s["kv_len"], s["table"], s["scale"])
    if kind == "batch":
        return kernels.attn_batch(s["q"], s["kc"], s["vc"], s["kv_len"], s["table"], s["scale"])
    return kernels.attn_shared(s["q"], s["kc"], s["vc"], s["kv_len"], s["table"], s["prefix_len"], s["prefix_table"], s["scale"])


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["kind"] == "append" else _plain_attend(state)


# ------------------------------------------------------------------ 64 bits, from the definitions
def _exact_append(s):
    n, ctx = _lengths(s)
    d, rot = s["d"], s["rot"]
    half = torch.arange(rot, device=DEV)
    if s["inter"]:
        partner, sign = half ^ 1, (half % 2 * 2 - 1).double()
    else:
        partner, sign = (half + rot // 2) % rot, torch.where(half < rot // 2, -1.0, 1.0).double()
    kc, vc = s["kc"].double(), s["vc"].double()
    outs, t = [], 0
    for b, (m, c) in enumerate(zip(n, ctx)):
        pos = torch.arange(c, c + m, device=DEV)
        cos, sin = s["cos"][c : c + m].double()[:, None], s["sin"][c : c + m].double()[:, None]
        new = []
        for x, w in ((s["q"], s["qn"]), (s["k"], s["kn"])):
            y = x[t : t + m].double()
            if w is not None:
                y = y / (y.square().sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
            z = y.clone()
            z[..., :rot] = y[..., :rot] * cos + sign * y[..., partner] * sin
            new.append(z)
        outs.append(new[0])
        pages = s["table"][b].long()[pos // s["page"]]
        kc[pages, :, pos % s["page"]] = new[1]
        vc[pages, :, pos % s["page"]] = s["v"][t : t + m].double()
        t += m
    return dict(q=torch.cat(outs), kc=kc, vc=vc)


def _exact_attend(s):
    n, ctx = _lengths(s)
    page, hk = s["page"], s["hk"]
    g = s["hq"] // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    t = 0
    for b, (m, c) in enumerate(zip(n, ctx)):
        rows = m if s["kind"] == "prompt" else 1
        at = [(s["table"][b].long(), m + c)]
        if s["kind"] == "shared":
            at.insert(0, (s["prefix_table"].long(), s["prefix"]))
        length = sum(x for _, x in at)
        for h in range(hk if length else 0):
            k, v = (torch.cat([c_[p[torch.arange(x, device=DEV) // page], h, torch.arange(x, device=DEV) % page] for p, x in at]).double()
                    for c_ in (s["kc"], s["vc"]))
            step = max(1, (1 << 27) // (g * length))
            for i in range(0, rows, step):
                e = min(rows, i + step)
                sc = torch.einsum("tgd,jd->tgj", s["q"][t + i : t + e, h * g : (h + 1) * g].double(), k) * s["scale"]
                seen = torch.arange(length, device=DEV)[None] <= torch.arange(length - rows + i, length - rows + e, device=DEV)[:, None]
                sc = torch.where(seen[:, None], sc, -math.inf)
                out[t + i : t + e, h * g : (h + 1) * g] = torch.einsum("tgj,jd->tgd", sc.softmax(-1), v)
        t += rows
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attend(s)


def work(case):
    n, ctx = _lengths(case)
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["kind"] == "append":
        T = sum(n)
        return dict(bytes=2 * T * (2 * (hq + 2 * hk) * d + 2 * case["rot"]), flops=T * (hq + hk) * (4 * d + 4 * case["rot"]))
    if case["kind"] == "prompt":
        kv, T = sum(a + b for a, b in zip(n, ctx) if a), sum(n)
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, ctx))
    else:
        kv, T = sum(n) + case.get("prefix", 0), case["B"]
        pairs = sum(n) + case["B"] * case.get("prefix", 0)
    return dict(bytes=2 * (2 * kv * hk * d + 2 * T * hq * d), flops=4 * pairs * hq * d)
