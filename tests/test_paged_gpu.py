"""The paged K/V cache (kv_append, attn_prompt, attn_batch, attn_shared) against plain restatements in 64 bits.

Bounds. u = finfo.eps / 2 is the most that one rounding to the type moves a value, relative to it.
kv_append: binary32 arithmetic, then one rounding: |got - ref| <= u |ref| (1 + d) + d S, S = |y cos| + |y' sin|, with
d = 2^-16 for binary32's share (a sum of 256 squares, a reciprocal square root, five products: below 300 roundings of
2^-24), plus the type's smallest step for values near zero.
Attention: o = sum p v / l. With A = sum softmax |v| the rounding of a weight to the type moves o by u A at most
(k_attn_rows; k_attn_flat splits weights in two terms, 2^-15 A), binary32 scores move a weight by e <= 2^-11
relative for the sizes here (D products of 2^-24 each, times |q||k| scale <= 2^7; exponents below 2^5 rounded at 2^-24)
and so o by 2 e A, and the result is rounded once: |got - ref| <= u |ref| + (w + 2^-10) A, w = u or 2^-15.
"""

import math

import numpy as np
import pytest
import torch

from wisp import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *shape, dtype=BF, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _tables(g, lens, page, spare=2, wider=1):
    """Random disjoint pages for `lens` positions each: (int32 [B, W], pages in all). Entries past a sequence's need: -1."""
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    t = torch.full((len(lens), max(need) + wider), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at : at + n]
        at += n
    return t, P


def _cache(g, P, hk, page, D, dtype, layout="hnd"):
    if layout == "hnd":
        return tuple(_rand(g, P, hk, page, D, dtype=dtype) for _ in range(2))
    if layout == "nhd":  # rows of all heads together: [P, page, hk, D] seen as [P, hk, page, D]
        return tuple(_rand(g, P, page, hk, D, dtype=dtype).transpose(1, 2) for _ in range(2))
    wide = _rand(g, P, 2, hk, page + 3, D + 8, dtype=dtype)  # keys and values interleaved, gaps between rows and heads
    return wide[:, 0, :, :page, :D], wide[:, 1, :, :page, :D]


def _pages_of(cache, row, n):
    """[Hk, n, D] in 64 bits: the first n positions of the sequence whose table row is given."""
    page = cache.shape[2]
    out = [cache[int(row[p // page]), :, p % page].double() for p in range(0, n)] if n < 64 else None
    if out is not None:
        return torch.stack(out, 1) if out else cache.new_zeros((cache.shape[1], 0, cache.shape[3]), dtype=torch.float64)
    idx = row[: -(-n // page)].long()
    return cache[idx].double().transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n]


def _attend(q, k, v, scale, lims):
    """q [n, Hq, D] against k, v [Hk, L, D], row i over positions <= lims[i]: (o, A) [n, Hq, D] in 64 bits."""
    n, hq, D = q.shape
    G = hq // k.shape[0]
    o = torch.zeros((n, hq, D), dtype=torch.float64, device=DEV)
    A = torch.zeros_like(o)
    for i, lim in enumerate(lims):
        if lim < 0:
            continue
        kk, vv = k[:, : lim + 1].repeat_interleave(G, 0), v[:, : lim + 1].repeat_interleave(G, 0)
        s = (kk * q[i].double()[:, None]).sum(-1) * scale
        p = (s - s.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
        o[i] = (p[..., None] * vv).sum(1)
        A[i] = (p[..., None] * vv.abs()).sum(1)
    return o, A


def _check(got, ref, A, dtype, flat, what=""):
    u = torch.finfo(dtype).eps / 2
    w = 2.0**-15 if flat else u
    tol = u * ref.abs() + (w + 2.0**-10) * A + torch.finfo(dtype).smallest_normal * 2.0**-8
    err = (got.double() - ref).abs()
    assert torch.isfinite(got.double()).all(), what
    assert (err <= tol).all(), (what, (err / tol.clamp_min(1e-300)).max().item())


# ------------------------------------------------------------------ kv_append
def _rope(rng_g, rows, rot, dtype, inter, cs32):
    inv = 1.0 / (1e4 ** (torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot))
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * inv
    ang = ang.repeat_interleave(2, 1) if inter else torch.cat([ang, ang], 1)
    t = torch.float32 if cs32 else dtype
    return ang.cos().to(t), ang.sin().to(t)


def _append_ref(x, w, eps, cos, sin, inter):
    """(out, S) of heads x [h, D] of one token in 64 bits."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    R = cos.numel()
    r = y[:, :R]
    if inter:
        t = torch.stack([-r[:, 1::2], r[:, 0::2]], -1).reshape(r.shape)
    else:
        t = torch.cat([-r[:, R // 2 :], r[:, : R // 2]], -1)
    out, S = y.clone(), y.abs().clone()
    out[:, :R] = r * cos.double() + t * sin.double()
    S[:, :R] = (r * cos.double()).abs() + (t * sin.double()).abs()
    return out, S


def _check_append(got, ref, S, dtype):
    u, d = torch.finfo(dtype).eps / 2, 2.0**-16
    tol = u * ref.abs() * (1 + d) + d * S + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (err / tol).max().item()


APPEND = [
    # dtype, hq, hk, D, rot, inter, norm, cs32, page, layout, new tokens, cached before
    (BF, 32, 4, 128, 128, False, True, False, 64, "hnd", [5, 1, 70], [0, 99, 64]),
    (BF, 8, 8, 128, 128, True, True, True, 16, "nhd", [1, 0, 33], [15, 0, 3]),
    (HF, 64, 8, 64, 64, False, False, False, 32, "hnd", [1, 1, 1, 1], [0, 31, 32, 500]),
    (HF, 16, 2, 256, 64, False, True, True, 128, "gaps", [17, 2], [0, 126]),
    (BF, 7, 1, 64, 16, True, True, False, 16, "gaps", [3, 20], [4, 0]),
    (HF, 2, 2, 256, 256, True, False, False, 16, "nhd", [2], [7]),
    (BF, 5, 5, 128, 32, False, False, True, 256, "hnd", [300], [0]),
    (HF, 28, 4, 128, 112, False, True, False, 64, "hnd", [0, 9, 0], [0, 60, 12]),
]


@pytest.mark.parametrize("case", APPEND, ids=[str(i) for i in range(len(APPEND))])
@pytest.mark.parametrize("fused", [True, False])
def test_append(case, fused):
    dtype, hq, hk, D, rot, inter, norm, cs32, page, layout, new, ctx = case
    g = _gen(hq * D + len(new))
    lens = [a + b for a, b in zip(new, ctx)]
    table, P = _tables(g, lens, page)
    kc, vc = _cache(g, P, hk, page, D, dtype, layout)
    k0, v0 = kc.clone(), vc.clone()
    T, tail = sum(new), 3
    if fused:  # one projection's output, with rows that belong to no sequence behind the last
        qkv = _rand(g, T + tail, hq + 2 * hk, D, dtype=dtype)
        q, k, v = qkv[:, :hq], qkv[:, hq : hq + hk], qkv[:, hq + hk :]
    else:  # heads first in memory
        q, k, v = (_rand(g, h, T + tail, D, dtype=dtype).transpose(0, 1) for h in (hq, hk, hk))
    qn, kn = (_rand(g, D, dtype=dtype, std=0.2) + 1 for _ in range(2)) if norm else (None, None)
    cos, sin = _rope(g, max(lens) + 1, rot, dtype, inter, cs32)
    qo = torch.full((T + tail, hq, D), 7.0, dtype=dtype, device=DEV)
    cu = _i32(np.cumsum([0] + new).tolist())
    got = kernels.kv_append(q, k, v, cos, sin, cu, _i32(lens), table, kc, vc, qn, kn, 1e-6, inter, qo)
    torch.cuda.synchronize()
    assert got is qo and (qo[T:] == 7.0).all()
    t = 0
    for b, n in enumerate(new):
        for j in range(n):
            p = ctx[b] + j
            ref, S = _append_ref(q[t], qn, 1e-6, cos[p], sin[p], inter)
            _check_append(qo[t], ref, S, dtype)
            at = int(table[b, p // page]), slice(None), p % page
            ref, S = _append_ref(k[t], kn, 1e-6, cos[p], sin[p], inter)
            _check_append(kc[at], ref, S, dtype)
            assert torch.equal(vc[at], v[t])
            k0[at], v0[at] = kc[at], vc[at]
            t += 1
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # every other row of the cache as it was


def test_append_without_sequences_or_tokens():
    g = _gen(1)
    kc, vc = _cache(g, 2, 2, 16, 64, BF)
    k0 = kc.clone()
    cos, sin = _rope(g, 8, 64, BF, False, False)
    q, k = _rand(g, 0, 4, 64), _rand(g, 0, 2, 64)
    out = kernels.kv_append(q, k, k, cos, sin, _i32([0, 0]), _i32([0]), _i32([[0]]), kc, vc)
    assert out.shape == (0, 4, 64)
    q, k = _rand(g, 3, 4, 64), _rand(g, 3, 2, 64)
    qo = torch.zeros_like(q)
    kernels.kv_append(q, k, k, cos, sin, _i32([0, 0]), _i32([0]), _i32([[0]]), kc, vc, qo=qo)
    assert torch.equal(kc, k0) and (qo == 0).all()


def test_append_where_there_is_no_place_stores_nothing():
    """Bad page ids, positions past the table, before 0 and past cos: NaN in the token's q, nothing stored, others right."""
    g = _gen(2)
    hq, hk, D, page = 4, 2, 128, 16
    kc, vc = _cache(g, 4, hk, page, D, BF)
    k0, v0 = kc.clone(), vc.clone()
    cos, sin = _rope(g, 40, D, BF, False, False)
    table = _i32([[0, 1], [9, 2], [-1, 3], [3, 3]])
    new, lens = [2, 20, 3, 20], [2, 20, 1, 45]
    q, k, v = (_rand(g, sum(new), h, D) for h in (hq, hk, hk))
    qo = kernels.kv_append(q, k, v, cos, sin, _i32(np.cumsum([0] + new).tolist()), _i32(lens), table, kc, vc)
    torch.cuda.synchronize()
    t = 0
    for b, n in enumerate(new):
        for j in range(n):
            p = lens[b] - n + j
            ok = 0 <= p < 32 and 0 <= int(table[b, p // page]) < 4
            if ok:
                at = int(table[b, p // page]), slice(None), p % page
                assert torch.isfinite(qo[t].float()).all()
                k0[at], v0[at] = kc[at], v[t]
            else:
                assert torch.isnan(qo[t].float()).all(), (b, j)
            t += 1
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_append_of_one_token_agrees_with_the_decoder_step():
    """The same token through dl_qk_rope, which rounds to bf16 after the norm and after the weight as the modules do: two
    more roundings of u each, of y and of its partner: 2 u S (1 + u) more than kv_append's bound."""
    g = _gen(3)
    hq, hk, D, tmax, pos = 32, 4, 128, 128, 77
    qkv = _rand(g, hq + 2 * hk, D)
    qn, kn = _rand(g, D, std=0.2) + 1, _rand(g, D, std=0.2) + 1
    cos, sin = _rope(g, tmax, D, BF, False, False)
    a, b = (torch.zeros(1, hk, tmax, D, dtype=BF, device=DEV) for _ in range(2))
    qo = torch.empty(hq * D, dtype=BF, device=DEV)
    kernels.dl_qk_rope(qkv.view(-1), qn, kn, 1e-6, cos, sin, torch.tensor([pos], device=DEV), hq, hk, D, a, b, qo)
    # the static cache as pages of 64
    kc, vc = (torch.zeros(hk, tmax // 64, 64, D, dtype=BF, device=DEV).transpose(0, 1) for _ in range(2))
    x = qkv.view(1, -1, D)
    got = kernels.kv_append(x[:, :hq], x[:, hq : hq + hk], x[:, hq + hk :], cos, sin, _i32([0, 1]), _i32([pos + 1]),
                            _i32([[0, 1]]), kc, vc, qn, kn)
    u = 2.0**-8
    for mine, theirs, h, w in ((got[0], qo.view(hq, D), qkv[:hq], qn), (kc[pos // 64, :, pos % 64], a[0, :, pos], qkv[hq : hq + hk], kn)):
        ref, S = _append_ref(h, w, 1e-6, cos[pos], sin[pos], False)
        _check_append(mine, ref, S, BF)
        assert ((mine.double() - theirs.double()).abs() <= 2 * u * ref.abs() + 2 * u * S * (1 + 4 * u)).all()
    assert torch.equal(vc[pos // 64, :, pos % 64], b[0, :, pos])


# ------------------------------------------------------------------ attn_prompt
def _prompt(seed, dtype, hq, hk, D, page, new, ctx, layout="hnd", wider=1, scale=None, qstd=1.0):
    g = _gen(seed)
    lens = [a + b for a, b in zip(new, ctx)]
    table, P = _tables(g, [max(n, 0) for n in lens], page, wider=wider)
    kc, vc = _cache(g, P, hk, page, D, dtype, layout)
    q = _rand(g, sum(new), hq, D, dtype=dtype, std=qstd)
    return dict(q=q, kc=kc, vc=vc, cu=_i32(np.cumsum([0] + new).tolist()), kv_len=_i32(lens), table=table,
                scale=D**-0.5 if scale is None else scale)


def _prompt_ref(s, new, ctx):
    o, A, t = [], [], 0
    for b, n in enumerate(new):
        L = max(n + ctx[b], 0)
        k, v = _pages_of(s["kc"], s["table"][b], L), _pages_of(s["vc"], s["table"][b], L)
        r = _attend(s["q"][t : t + n], k, v, s["scale"], [ctx[b] + j for j in range(n)])
        o.append(r[0])
        A.append(r[1])
        t += n
    return torch.cat(o), torch.cat(A)


PROMPT = [
    # dtype, hq, hk, D, page, layout, new tokens, cached before (negative: leading rows attend nothing)
    (BF, 32, 4, 128, 64, "hnd", [1], [0]),
    (BF, 32, 4, 128, 64, "hnd", [61, 1, 0, 130], [0, 63, 5, 0]),
    (BF, 8, 8, 128, 16, "nhd", [257, 3], [0, 1000]),
    (HF, 64, 8, 64, 32, "hnd", [100, 31], [77, 0]),
    (HF, 16, 2, 256, 128, "gaps", [65, 17], [0, 300]),
    (BF, 16, 1, 256, 16, "hnd", [40], [3]),
    (BF, 28, 4, 128, 256, "gaps", [75, 64], [64, 0]),
    (HF, 5, 1, 64, 16, "nhd", [90, 2, 63], [0, 40, 1]),
    (BF, 4, 4, 64, 64, "hnd", [300], [0]),
    (BF, 40, 8, 128, 64, "hnd", [10, 12], [-4, -12]),
    (HF, 24, 1, 128, 64, "hnd", [33], [64]),
    (BF, 64, 16, 64, 64, "hnd", [700, 0, 641], [0, 10, 3]),  # many rows of 64: four waves a workgroup
    (HF, 36, 18, 64, 32, "nhd", [2300], [0]),
]


@pytest.mark.parametrize("case", PROMPT, ids=[str(i) for i in range(len(PROMPT))])
def test_prompt(case):
    dtype, hq, hk, D, page, layout, new, ctx = case
    s = _prompt(hq + D + len(new), dtype, hq, hk, D, page, new, ctx, layout)
    ref, A = _prompt_ref(s, new, ctx)
    got = kernels.attn_prompt(**s)
    _check(got, ref, A, dtype, False)


@pytest.mark.parametrize("dtype,hq,hk,D,new,ctx", [
    (BF, 32, 4, 128, [3, 9], [5000, 700]), (HF, 64, 8, 64, [20], [9000]), (BF, 16, 2, 256, [1, 1, 2], [3000, 0, 64]),
    (BF, 8, 8, 128, [1], [4111])])
def test_prompt_of_few_tokens_behind_a_long_context(dtype, hq, hk, D, new, ctx):
    """Positions cut into parts that are joined; the first sequence's and the short ones' tiles are cut differently."""
    s = _prompt(9 + D, dtype, hq, hk, D, 64, new, ctx, wider=40)
    ref, A = _prompt_ref(s, new, ctx)
    _check(kernels.attn_prompt(**s), ref, A, dtype, False)


def test_prompt_of_large_scores():
    """Scores of several hundred: the reference of the running sum moves far and often."""
    for dtype in (BF, HF):
        s = _prompt(4, dtype, 8, 2, 64, 32, [150], [200], qstd=30.0)
        ref, A = _prompt_ref(s, [150], [200])
        got = kernels.attn_prompt(**s)
        u = torch.finfo(dtype).eps / 2
        # |q||k| scale <= 30 * 64 * 0.125 * 8 ~ 2^11, products in binary32: weights move by 64 * 2^-24 * 2^11 = 2^-7
        tol = u * ref.abs() + (u + 2.0**-6) * A + 1e-6
        assert ((got.double() - ref).abs() <= tol).all()


def test_prompt_strided_q_and_rows_behind_the_last_sequence():
    g = _gen(8)
    s = _prompt(8, BF, 8, 2, 128, 16, [20, 30], [0, 5])
    want = kernels.attn_prompt(**s)
    wide = _rand(g, 60, 12, 128)
    wide[:50, 2:10] = s["q"]
    out = torch.full((60, 8, 128), 3.0, dtype=BF, device=DEV)
    got = kernels.attn_prompt(**dict(s, q=wide[:, 2:10]), out=out)
    assert torch.equal(got[:50], want) and (out[50:] == 3.0).all()
    odd = torch.empty(50 * 8 * 128 + 4, dtype=BF, device=DEV)[4:].view(50, 8, 128)  # not 16-byte aligned: copied
    odd.copy_(s["q"])
    assert torch.equal(kernels.attn_prompt(**dict(s, q=odd)), want)


def _poison(s, lens, value):
    """Every cache row that holds no position of a sequence set to `value`."""
    page = s["kc"].shape[2]
    used = torch.zeros(s["kc"].shape[0], page, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for p in range(n):
            used[int(s["table"][b, p // page]), p % page] = True
    for c in (s["kc"], s["vc"]):
        c.transpose(1, 2)[~used] = value


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_lies_behind_a_sequence_does_not_matter(D, value):
    new, ctx = [40, 7, 130], [3, 0, 20]
    lens = [a + b for a, b in zip(new, ctx)]
    s = _prompt(11, BF, 8, 2, D, 32, new, ctx)
    want = kernels.attn_prompt(**s)
    b_args = dict(q=s["q"][:3].contiguous(), kc=s["kc"], vc=s["vc"], kv_len=s["kv_len"], table=s["table"], scale=s["scale"])
    want_b = kernels.attn_batch(**b_args)
    pre = dict(prefix_len=_i32([lens[2]]), prefix_table=s["table"][2].contiguous())
    want_s = kernels.attn_shared(**b_args, **pre)
    _poison(s, lens, value)
    assert torch.equal(kernels.attn_prompt(**s), want)
    assert torch.equal(kernels.attn_batch(**b_args), want_b)
    assert torch.equal(kernels.attn_shared(**b_args, **pre), want_s)


@pytest.mark.parametrize("dtype,D,hq,hk", [(BF, 128, 8, 2), (HF, 64, 4, 4), (BF, 256, 8, 1)])
def test_non_finite_values_reach_only_the_rows_that_attend_them(dtype, D, hq, hk):
    """inf, -inf and NaN in V, and NaN in K, at positions in the middle of the prompt: earlier rows are as without them."""
    new, ctx = [150], [10]
    for value, where in ((math.inf, "v"), (-math.inf, "v"), (math.nan, "v"), (math.nan, "k")):
        s = _prompt(12, dtype, hq, hk, D, 16, new, ctx)
        want = kernels.attn_prompt(**s)
        row, at = s["table"][0], 101  # position 101: token 91
        cache = s["vc"] if where == "v" else s["kc"]
        cache[int(row[at // 16]), :, at % 16, 5] = value
        got = kernels.attn_prompt(**s)
        assert torch.equal(got[:91], want[:91])
        hit = got[91:, :, 5] if where == "v" else got[91:]
        if math.isnan(value):
            assert torch.isnan(hit.float()).all()
        else:
            assert (hit == value).all()
        if where == "v":
            rest = [d for d in range(D) if d != 5]
            u = torch.finfo(dtype).eps / 2
            assert ((got[91:][..., rest].double() - want[91:][..., rest].double()).abs() <= 2 * u * 4).all()


@pytest.mark.parametrize("bad", [-1, 1 << 30, 99])
def test_a_bad_page_gives_nan_for_its_sequence_only(bad):
    new, ctx = [70, 40], [100, 30]
    s = _prompt(13, BF, 8, 2, 128, 16, new, ctx)
    args = dict(q=s["q"][:2].contiguous(), kc=s["kc"], vc=s["vc"], kv_len=s["kv_len"], table=s["table"], scale=s["scale"])
    want, want_b = kernels.attn_prompt(**s), kernels.attn_batch(**args)
    s["table"][0, 6] = bad  # positions 96 .. 111: every token of the first sequence attends it
    got, got_b = kernels.attn_prompt(**s), kernels.attn_batch(**args)
    assert torch.isnan(got[:70].float()).all() and torch.equal(got[70:], want[70:])
    assert torch.isnan(got_b[0].float()).all() and torch.equal(got_b[1], want_b[1])
    pre = kernels.attn_shared(**args, prefix_len=_i32([64]), prefix_table=_i32([0, 1, bad, 3]))
    assert torch.isnan(pre.float()).all()


def test_a_length_past_the_table_gives_nan():
    s = _prompt(14, BF, 8, 2, 128, 16, [5, 5], [20, 3], wider=0)
    args = dict(q=s["q"][:2].contiguous(), kc=s["kc"], vc=s["vc"], table=s["table"], scale=s["scale"])
    W = s["table"].shape[1] * 16
    for n in (W + 1, 2**31 - 1):
        got = kernels.attn_prompt(**dict(s, kv_len=_i32([n, 8])))
        assert torch.isnan(got[:5].float()).all() and torch.isfinite(got[5:].float()).all()
        got = kernels.attn_batch(**args, kv_len=_i32([n, 8]))
        assert torch.isnan(got[0].float()).all() and torch.isfinite(got[1].float()).all()
    got = kernels.attn_batch(**args, kv_len=_i32([-5, 8]))
    assert (got[0] == 0).all() and torch.isfinite(got[1].float()).all()


# ------------------------------------------------------------------ attn_batch and attn_shared
def _batch(seed, dtype, hq, hk, D, page, lens, layout="hnd", prefix=None, qstd=1.0):
    g = _gen(seed)
    table, P = _tables(g, lens + ([prefix] if prefix else []), page)
    kc, vc = _cache(g, P, hk, page, D, dtype, layout)
    s = dict(q=_rand(g, len(lens), hq, D, dtype=dtype, std=qstd), kc=kc, vc=vc, kv_len=_i32(lens), scale=D**-0.5,
             table=table[: len(lens)].contiguous())
    if prefix is not None:
        s.update(prefix_len=_i32([prefix]), prefix_table=table[-1].contiguous())
    return s


def _batch_ref(s, lens, prefix=0):
    o, A = [], []
    for b, n in enumerate(lens):
        k, v = _pages_of(s["kc"], s["table"][b], n), _pages_of(s["vc"], s["table"][b], n)
        if prefix:
            k = torch.cat([_pages_of(s["kc"], s["prefix_table"], prefix), k], 1)
            v = torch.cat([_pages_of(s["vc"], s["prefix_table"], prefix), v], 1)
        r = _attend(s["q"][b : b + 1], k, v, s["scale"], [k.shape[1] - 1])
        o.append(r[0])
        A.append(r[1])
    return torch.cat(o), torch.cat(A)


BATCH = [
    (BF, 32, 4, 128, 64, "hnd", [1]),
    (BF, 32, 4, 128, 64, "hnd", [0, 1, 2, 31, 32, 33, 127, 128, 129, 1000]),
    (HF, 64, 8, 64, 32, "nhd", [5000, 3, 0, 640]),
    (BF, 16, 2, 256, 16, "gaps", [300, 77]),
    (HF, 20, 1, 128, 64, "hnd", [50, 400]),
    (BF, 32, 1, 64, 64, "hnd", [129, 4]),
    (BF, 28, 4, 128, 256, "hnd", [900, 1, 513]),
    (HF, 3, 3, 256, 32, "hnd", [64, 65, 66]),
    (BF, 8, 2, 128, 16, "hnd", [(37 * i) % 300 for i in range(150)]),
    (BF, 8, 1, 64, 64, "hnd", [70000]),
    (BF, 32, 4, 128, 64, "hnd", [200, 0, 512, 7]),  # short tables: taken whole
    (HF, 20, 1, 64, 16, "nhd", [(13 * i) % 500 for i in range(130)]),
    (HF, 16, 2, 256, 64, "hnd", [1025, 0, 3000]),
]


@pytest.mark.parametrize("case", BATCH, ids=[str(i) for i in range(len(BATCH))])
def test_batch(case):
    dtype, hq, hk, D, page, layout, lens = case
    s = _batch(hq + D, dtype, hq, hk, D, page, lens, layout)
    ref, A = _batch_ref(s, lens)
    _check(kernels.attn_batch(**s), ref, A, dtype, True)


SHARED = [
    (BF, 32, 4, 128, 64, "hnd", 1531, [1, 200, 0, 65]),
    (BF, 32, 4, 128, 64, "hnd", 1, [0]),
    (HF, 64, 8, 64, 32, "hnd", 700, [3] * 9),
    (BF, 16, 2, 256, 16, "nhd", 333, [20, 1]),
    (HF, 40, 8, 128, 128, "gaps", 64, [(11 * i) % 130 for i in range(70)]),
    (BF, 7, 1, 128, 64, "hnd", 5000, [10, 0, 300]),
    (BF, 32, 4, 128, 64, "hnd", 900, [1500, 0, 3]),  # own tables past what is taken whole
    (HF, 20, 1, 64, 32, "hnd", 9000, [2000, 5]),
    (HF, 16, 2, 256, 16, "hnd", 2000, [1100, 0, 64, 9]),
]


@pytest.mark.parametrize("case", SHARED, ids=[str(i) for i in range(len(SHARED))])
def test_shared(case):
    dtype, hq, hk, D, page, layout, prefix, lens = case
    s = _batch(hq + D + 1, dtype, hq, hk, D, page, lens, layout, prefix)
    ref, A = _batch_ref(s, lens, prefix)
    _check(kernels.attn_shared(**s), ref, A, dtype, False)


def test_an_empty_prefix_is_attn_batch():
    s = _batch(21, BF, 32, 4, 128, 64, [40, 0, 500], prefix=64)
    s["prefix_len"] = _i32([0])
    own = {k: v for k, v in s.items() if not k.startswith("prefix")}
    a, b = kernels.attn_shared(**s), kernels.attn_batch(**own)
    u = 2.0**-8
    assert ((a.double() - b.double()).abs() <= 2 * u * b.double().abs() + 1e-6).all() and (a[1] == 0).all()


def test_attn_batch_of_one_agrees_with_attn_decode():
    g = _gen(22)
    hq, hk, D, tmax, pos = 32, 4, 128, 512, 300
    kc, vc = _rand(g, 1, hk, tmax, D), _rand(g, 1, hk, tmax, D)
    q = _rand(g, 1, hq, D)
    want = kernels.attn_decode(q[0], kc, vc, torch.tensor([pos], device=DEV), D**-0.5).view(1, hq, D)
    pages = [c[0].view(hk, tmax // 64, 64, D).transpose(0, 1) for c in (kc, vc)]
    got = kernels.attn_batch(q, *pages, _i32([pos + 1]), torch.arange(tmax // 64, dtype=torch.int32, device=DEV)[None], D**-0.5)
    # both carry binary32 sums and one rounding: a value near a rounding border may fall on either side
    assert ((got.double() - want.double()).abs() <= 2.0**-7 * want.double().abs() + 1e-5).all()
    assert (got != want).float().mean().item() < 0.02


def test_a_cache_past_four_gigabytes():
    """Page offsets past 2^32 bytes, in both directions of a table."""
    hk, page, D = 4, 256, 128
    P = (9 << 30) // 2 // (hk * page * D * 2)  # 4.5 GiB a cache
    g = _gen(23)
    kc = torch.empty((P, hk, page, D), dtype=BF, device=DEV)
    vc = torch.empty_like(kc)
    ids = [P - 1, 0, P - 2, 1, P // 2]
    for c in (kc, vc):
        for i in ids:
            c[i] = _rand(g, hk, page, D)
    lens, new = [700, 500], [30, 20]
    table = _i32([ids[:3], [ids[4], ids[3], 0]])
    q = _rand(g, 2, 32, D)
    s = dict(q=q, kc=kc, vc=vc, kv_len=_i32(lens), table=table, scale=D**-0.5)
    ref, A = _batch_ref(s, lens)
    _check(kernels.attn_batch(**s), ref, A, BF, True)
    q = _rand(g, sum(new), 32, D)
    s = dict(q=q, kc=kc, vc=vc, cu=_i32([0, 30, 50]), kv_len=_i32(lens), table=table, scale=D**-0.5)
    ref, A = _prompt_ref(s, new, [670, 480])
    _check(kernels.attn_prompt(**s), ref, A, BF, False)
    k, v = _rand(g, 50, hk, D), _rand(g, 50, hk, D)
    cos, sin = torch.ones(700, D, device=DEV), torch.zeros(700, D, device=DEV)
    kernels.kv_append(q, k, v, cos, sin, s["cu"], s["kv_len"], table, kc, vc)
    got = _pages_of(kc, table[0], 700)[:, 670:], _pages_of(vc, table[1], 500)[:, 480:]
    assert torch.equal(got[0], k[:30].double().transpose(0, 1)) and torch.equal(got[1], v[30:].double().transpose(0, 1))


# ------------------------------------------------------------------ together, as a server runs them
def test_prompts_then_steps_as_a_server_runs_them():
    """Three requests: their prompts appended and attended in two chunks, then five decode steps, then four samples of the
    third behind its prompt as a shared prefix; every output against attention in 64 bits over the keys and values that
    the cache holds, and those against their own restatement."""
    g = _gen(30)
    hq, hk, D, page, W = 16, 4, 128, 32, 12
    table = torch.randperm(3 * W, generator=g, device=DEV).to(torch.int32).view(3, W)
    kc, vc = (torch.full((3 * W, hk, page, D), math.nan, dtype=BF, device=DEV) for _ in range(2))
    cos, sin = _rope(g, 400, D, BF, False, False)
    qn, kn = _rand(g, D, std=0.1) + 1, _rand(g, D, std=0.1) + 1
    done = [0, 0, 0]
    keys = [[], [], []]
    for new in ([70, 33, 200], [5, 0, 90], [1, 1, 1], [1, 1, 1], [1, 0, 1], [1, 1, 1]):
        T = sum(new)
        qkv = _rand(g, T, hq + 2 * hk, D)
        done = [a + b for a, b in zip(done, new)]
        cu, kv_len = _i32(np.cumsum([0] + new).tolist()), _i32(done)
        q = kernels.kv_append(qkv[:, :hq], qkv[:, hq : hq + hk], qkv[:, hq + hk :], cos, sin, cu, kv_len, table, kc, vc, qn, kn)
        t = 0
        for b, n in enumerate(new):
            keys[b] += [_append_ref(qkv[t + j, hq : hq + hk], kn, 1e-6, cos[done[b] - n + j], sin[done[b] - n + j], False)
                        for j in range(n)]
            t += n
        s = dict(q=q, kc=kc, vc=vc, cu=cu, kv_len=kv_len, table=table, scale=D**-0.5)
        ref, A = _prompt_ref(s, new, [a - b for a, b in zip(done, new)])
        _check(kernels.attn_prompt(**s), ref, A, BF, False)
        if new == [1, 1, 1]:
            _check(kernels.attn_batch(q, kc, vc, kv_len, table, D**-0.5), ref, A, BF, True)
    for b in range(3):
        got = _pages_of(kc, table[b], done[b]).transpose(0, 1)
        _check_append(got, torch.stack([r for r, _ in keys[b]]), torch.stack([S for _, S in keys[b]]), BF)
    n, own = 4, table[:1, :4].reshape(4, 1).contiguous()
    s = dict(q=_rand(g, n, hq, D), kc=kc, vc=vc, kv_len=_i32([0] * n), table=own, scale=D**-0.5, prefix_len=_i32([done[2]]),
             prefix_table=table[2].contiguous())
    ref, A = _batch_ref(s, [0] * n, done[2])
    _check(kernels.attn_shared(**s), ref, A, BF, False)


def test_captured_calls_follow_the_lengths_and_pages():
    """append, prompt, batch and shared in two graphs (each with its own workspaces), replayed in turn with new lengths,
    tables and inputs and eager work between: bit for bit the eager calls."""
    g = _gen(31)
    hq, hk, D, page, B, W, T = 8, 2, 128, 16, 3, 30, 24
    kc, vc = _cache(g, B * W + 4, hk, page, D, BF)
    cos, sin = _rope(g, W * page, D, BF, False, False)
    st = dict(qkv=_rand(g, T, hq + 2 * hk, D), cu=_i32([0, 8, 16, 24]), kv_len=_i32([100, 200, 300]),
              table=torch.arange(B * W, dtype=torch.int32, device=DEV).view(B, W), plen=_i32([33]),
              ptable=_i32([B * W, B * W + 1, B * W + 2]))

    def calls(x, kc, vc):
        q = kernels.kv_append(x["qkv"][:, :hq], x["qkv"][:, hq : hq + hk], x["qkv"][:, hq + hk :], cos, sin, x["cu"],
                              x["kv_len"], x["table"], kc, vc)
        a = kernels.attn_prompt(q, kc, vc, x["cu"], x["kv_len"], x["table"], 0.1)
        b = kernels.attn_batch(q[:B], kc, vc, x["kv_len"], x["table"], 0.1)
        c = kernels.attn_shared(q[:B], kc, vc, x["kv_len"], x["table"], x["plen"], x["ptable"], 0.1)
        return q, a, b, c

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(st, kc, vc)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = calls(st, kc, vc)
        graphs.append((gr, out))
    rng = np.random.default_rng(5)
    for it in range(5):
        new = rng.integers(0, 9, B)
        lens = new + rng.integers(0, W * page - 10, B)
        st["qkv"].copy_(_rand(g, T, hq + 2 * hk, D))
        st["cu"].copy_(_i32(np.cumsum([0] + new.tolist()).tolist()))
        st["kv_len"].copy_(_i32(lens.tolist()))
        st["table"].copy_(torch.randperm(B * W, generator=g, device=DEV).view(B, W))
        st["plen"].copy_(_i32([int(rng.integers(0, 49))]))
        n = int(new.sum())
        k1, v1 = kc.clone(), vc.clone()
        want = calls(st, k1, v1)
        for gr, out in graphs:
            for o in out:
                o.zero_()
            gr.replay()
            torch.cuda.synchronize()
            for i, (o, w) in enumerate(zip(out, want)):
                m = n if i < 2 else (min(n, B))  # (rows of q behind the last sequence are undefined)
                assert torch.equal(o[:m], w[:m]), (it, i)
            assert torch.equal(kc, k1) and torch.equal(vc, v1)
        torch.randn(64, device=DEV).sum().item()


def test_another_stream_and_repeated_calls():
    s = _batch(33, BF, 32, 4, 128, 64, [3000, 17, 900])
    p = _prompt(34, BF, 32, 4, 128, 64, [5, 3], [4000, 90])
    want, want_p = kernels.attn_batch(**s), kernels.attn_prompt(**p)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append((kernels.attn_batch(**s), kernels.attn_prompt(**p)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want) and torch.equal(b, want_p)


def _heads(seed, T, hq, hk, D, dtype):
    g = _gen(seed)
    x = _rand(g, T, hq + 2 * hk, D, dtype=dtype)
    return x[:, :hq], x[:, hq : hq + hk], x[:, hq + hk :]


@pytest.mark.parametrize("dtype,D,inter", [(BF, 128, False), (HF, 64, True)])
def test_append_of_many_tokens_is_that_of_its_slices(dtype, D, inter):
    """However a call's heads are dealt out to waves, which follows its number of tokens, a token's result is the same."""
    T, hq, hk = 6300, 32, 4
    g = _gen(40)
    table, P = _tables(g, [T], 64)
    q, k, v = _heads(41, T, hq, hk, D, dtype)
    cos, sin = _rope(g, T, D, dtype, inter, True)
    w = [_rand(g, D, dtype=dtype) for _ in range(2)]
    caches = [_cache(_gen(42), P, hk, 64, D, dtype) for _ in range(2)]
    whole = kernels.kv_append(q, k, v, cos, sin, _i32([0, T]), _i32([T]), table, *caches[0], *w, interleaved=inter)
    parts = []
    for lo, hi in [(0, 1), (1, 700), (700, 4900), (4900, T)]:
        parts.append(kernels.kv_append(q[lo:hi], k[lo:hi], v[lo:hi], cos, sin, _i32([0, hi - lo]), _i32([hi]), table, *caches[1],
                                       *w, interleaved=inter))
    assert torch.equal(whole, torch.cat(parts))
    for a, b in zip(*caches):
        assert torch.equal(a, b)


def test_more_sequences_than_lanes():
    new = [(5 * i) % 4 for i in range(150)]
    ctx = [(29 * i) % 90 for i in range(150)]
    s = _prompt(43, BF, 8, 2, 128, 16, new, ctx)
    ref, A = _prompt_ref(s, new, ctx)
    _check(kernels.attn_prompt(**s), ref, A, BF, False)
    T = sum(new)
    q, k, v = _heads(44, T, 8, 2, 128, BF)
    cos, sin = _rope(_gen(45), 128, 128, BF, False, False)
    caches = [[t.clone() for t in (s["kc"], s["vc"])] for _ in range(2)]
    whole = kernels.kv_append(q, k, v, cos, sin, s["cu"], s["kv_len"], s["table"], *caches[0])
    parts, cu = [], s["cu"].tolist()
    for b in range(0, 150, 50):
        lo, hi = cu[b], cu[b + 50]
        parts.append(kernels.kv_append(q[lo:hi], k[lo:hi], v[lo:hi], cos, sin, s["cu"][b : b + 51] - lo, s["kv_len"][b : b + 50],
                                       s["table"][b : b + 50], *caches[1]))
    assert torch.equal(whole, torch.cat(parts))
    for a, b in zip(*caches):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,hq,hk", [(64, 20, 1), (128, 32, 4), (256, 8, 8)])
def test_results_over_their_queries(D, hq, hk):
    for new, ctx in [([70, 3], [200, 900]), ([1], [6000])]:
        p = _prompt(46, BF, hq, hk, D, 64, new, ctx)
        want = kernels.attn_prompt(**p)
        assert torch.equal(kernels.attn_prompt(**p, out=p["q"]), want) and torch.equal(p["q"], want)
    for prefix in (None, 700):
        for lens in ([300, 0, 40], [3000, 5]):
            s = _batch(47, BF, hq, hk, D, 64, lens, prefix=prefix)
            call = kernels.attn_shared if prefix else kernels.attn_batch
            want = call(**s)
            assert torch.equal(call(**s, out=s["q"]), want) and torch.equal(s["q"], want)
    g = _gen(48)
    q, k, v = (_rand(g, 40, h, D) for h in (hq, hk, hk))
    cos, sin = _rope(g, 40, D, BF, False, True)
    caches = [_cache(_gen(49), 1, hk, 64, D, BF) for _ in range(2)]
    args = [cos, sin, _i32([0, 40]), _i32([40]), _i32([[0]])]
    want = kernels.kv_append(q, k, v, *args, *caches[0])
    assert torch.equal(kernels.kv_append(q, k, v, *args, *caches[1], qo=q), want)


def test_the_same_pages_in_several_sequences():
    s = _batch(50, BF, 32, 4, 128, 64, [700, 700, 130])
    s["table"][1:] = s["table"][0]
    ref, A = _batch_ref(s, [700, 700, 130])
    _check(kernels.attn_batch(**s), ref, A, BF, True)
    p = _prompt(51, HF, 8, 2, 64, 32, [9, 40], [300, 64])
    p["table"][1] = p["table"][0]
    ref, A = _prompt_ref(p, [9, 40], [300, 64])
    _check(kernels.attn_prompt(**p), ref, A, HF, False)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(D):
    p = _prompt(52, BF, 8, 2, D, 64, [50], [170])
    ref, A = _prompt_ref(p, [50], [170])
    p["q"][17, 3, 5] = math.nan
    got = kernels.attn_prompt(**p)
    assert got[17, 3].isnan().all()
    got[17, 3], ref[17, 3] = 0, 0
    _check(got, ref, A, BF, False)
    s = _batch(53, BF, 8, 2, D, 64, [50, 900])
    ref, A = _batch_ref(s, [50, 900])
    s["q"][1, 6, 0] = math.nan
    got = kernels.attn_batch(**s)
    assert got[1, 6].isnan().all()
    got[1, 6], ref[1, 6] = 0, 0
    _check(got, ref, A, BF, True)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_whose_scores_are_all_minus_infinity_give_zeros(D):
    p = _prompt(54, BF, 8, 2, D, 64, [40], [100])
    p["q"][..., 0] = 1
    p["kc"][..., 0] = -math.inf
    assert (kernels.attn_prompt(**p) == 0).all()
    s = _batch(55, BF, 8, 2, D, 64, [40, 3000], prefix=300)
    s["q"][..., 0] = 1
    s["kc"][..., 0] = -math.inf
    assert (kernels.attn_shared(**s) == 0).all()
    del s["prefix_len"], s["prefix_table"]
    assert (kernels.attn_batch(**s) == 0).all()


@pytest.mark.parametrize("dtype,hq,hk,D", [(BF, 32, 4, 128), (HF, 20, 1, 64), (BF, 6, 2, 64), (HF, 16, 2, 256), (BF, 3, 3, 256)])
@pytest.mark.parametrize("lens,prefix", [([40, 3000, 700], None), ([300, 129, 0], None), ([40, 200, 700], 900), ([5, 1500, 33], 2100)])
def test_an_infinite_value_that_is_attended_gives_an_infinity(dtype, hq, hk, D, lens, prefix):
    """Weights are split in two terms, of which the second is often 0 or negative. Own positions and a prefix's, cut into pieces
    or taken whole; every other element as it is without the infinity, bit for bit."""
    call = kernels.attn_shared if prefix else kernels.attn_batch
    s = _batch(60, dtype, hq, hk, D, 32, lens, "nhd", prefix=prefix)
    want = call(**s)
    rows = [("table", 0, 17 % lens[0], [0]), ("table", 1, lens[1] - 1, [1])]
    if prefix:
        rows.append(("prefix", None, 515, [0, 1, 2]))
    for where, b, p, hit in rows:
        page = int(s["prefix_table"][p // 32] if where == "prefix" else s["table"][b, p // 32])
        for value in (math.inf, -math.inf, math.nan):
            vc = s["vc"].clone()
            vc[page, :, p % 32, 7] = value
            vc[page, :, p % 32, D - 1] = -value
            got = call(**dict(s, vc=vc))
            for d, v in ((7, value), (D - 1, -value)):
                x = got[hit][:, :, d]
                assert (x.isnan() if math.isnan(v) else x == v).all(), (where, value, d)
            rest = torch.ones_like(want, dtype=torch.bool)
            for h in hit:
                rest[h, :, 7] = rest[h, :, D - 1] = False
            assert torch.equal(got[rest], want[rest])
    vc = s["vc"].clone()  # both signs: NaN
    page = int(s["table"][1, 0])
    vc[page, :, 3, 7], vc[page, :, 5, 7] = math.inf, -math.inf
    got = call(**dict(s, vc=vc))
    assert got[1, :, 7].isnan().all() and torch.isfinite(got[1, :, :7].float()).all()


@pytest.mark.parametrize("dtype,D", [(HF, 64), (HF, 128), (HF, 256), (BF, 128)])
def test_an_infinite_value_of_a_small_weight_gives_an_infinity(dtype, D):
    """A weight of e^-30: 0 in float16, not in binary32. It is met in tiles that all rows attend and in others, before and
    after the large weights. One of e^-200 is 0 in binary32, too: there the result is only known not to be finite."""
    n, page = 700, 64
    kc, vc = torch.zeros(11, 1, page, D, dtype=dtype, device=DEV), _rand(_gen(61), 11, 1, page, D, dtype=dtype)
    table = torch.arange(11, dtype=torch.int32, device=DEV)[None]
    q = torch.zeros(n, 2, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    for p, gap in ((3, 30), (100, 30), (599, 30), (3, 200)):
        k, v = kc.clone(), vc.clone()
        k[p // page, 0, p % page, 0] = -gap
        v[p // page, 0, p % page, 9] = -math.inf
        a = kernels.attn_prompt(q, k, v, _i32([0, n]), _i32([n]), table, 1.0)
        b = kernels.attn_batch(q[:1], k, v, _i32([n]), table, 1.0)
        c = kernels.attn_shared(q[:1], k, v, _i32([60]), table[:, 10:].contiguous(), _i32([640]), table[0, :10].contiguous(), 1.0)
        hit = [a[p + 1 :, :, 9], b[..., 9], c[..., 9]]
        for x in hit:
            assert ((x == -math.inf) if gap == 30 else ~torch.isfinite(x.float())).all(), (p, gap)
        for x in (a, b, c):
            assert torch.isfinite(x[..., :9].float()).all() and torch.isfinite(x[..., 10:].float()).all()
        assert torch.isfinite(a[:p].float()).all()


def test_append_of_more_tokens_than_one_grid_dimension_holds():
    """2^26 + 5 tokens (four of a workgroup of 256 threads: past 2^32 threads), all but the last five at positions before 0:
    NaN in their rows; the last five are stored. One row of q, k and v is read for all."""
    T = (1 << 26) + 5
    g = _gen(62)
    x = _rand(g, 1, 1, 64)
    kc, vc = _cache(g, 1, 1, 16, 64, BF)
    v0 = vc.clone()
    cos, sin = _rope(g, 16, 64, BF, False, True)
    qo = torch.zeros(T, 1, 64, dtype=BF, device=DEV)
    rows = x.expand(T, 1, 64)
    kernels.kv_append(rows, rows, rows, cos, sin, _i32([0, T]), _i32([5]), _i32([[0]]), kc, vc, qo=qo)
    for i in range(0, T - 5, 1 << 23):
        assert qo[i : min(i + (1 << 23), T - 5)].isnan().all(), i
    for p in range(5):
        ref, S = _append_ref(x[0], None, 0.0, cos[p], sin[p], False)
        _check_append(qo[T - 5 + p], ref, S, BF)
        _check_append(kc[0, :, p], ref, S, BF)
        v0[0, :, p] = x[0]
    assert torch.equal(vc, v0)


def test_batch_of_more_rows_than_one_grid_dimension_holds():
    """2^24 rows (a workgroup of 256 threads each where records are joined: 2^32 threads): sequences without positions among
    short ones, and a last one long enough to be cut."""
    B, hq, hk, page, long = 1 << 14, 1024, 64, 2048, 300000
    g = _gen(63)
    W = -(-long // page)
    kc, vc = (_rand(g, 3, hk, page, 64) for _ in range(2))
    lens = [(7 * i) % 4 for i in range(B - 1)] + [long]
    table = torch.randint(0, 3, (B, W), generator=g, device=DEV, dtype=torch.int32)
    q = _rand(g, B, hq, 64)
    out = torch.full_like(q, 7.0)
    kernels.attn_batch(q, kc, vc, _i32(lens), table, 0.125, out=out)
    few = 4000
    some = kernels.attn_batch(q[:few], kc, vc, _i32(lens[:few]), table[:few].contiguous(), 0.125)
    assert torch.equal(out[:few], some)
    some = kernels.attn_batch(q[-few:-1], kc, vc, _i32(lens[-few:-1]), table[-few:-1].contiguous(), 0.125)
    assert torch.equal(out[-few:-1], some)
    empty = torch.tensor(lens, device=DEV) == 0
    assert (out[empty] == 0).all()
    heads = [0, 5, 63]
    k, v = (torch.cat([c[table[-1, w].long()][heads] for w in range(W)], 1)[:, :long].double() for c in (kc, vc))
    rows = torch.cat([q[-1:, 16 * h : 16 * h + 16] for h in heads], 1)
    p = (torch.matmul(rows.view(3, 16, 64).double(), k.transpose(1, 2).contiguous()) * 0.125).softmax(-1)
    ref, A = (torch.matmul(p, x).view(1, 48, 64) for x in (v, v.abs()))
    got = torch.cat([out[-1:, 16 * h : 16 * h + 16] for h in heads], 1)
    _check(got, ref, A, BF, True)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_an_odd_number_of_records(D):
    """7 query heads over one, 43 tiles of positions in 21 parts, one row: 147 records."""
    s = _prompt(64, BF, 7, 1, D, 64, [1], [2700], wider=0)
    assert s["table"].shape[1] == 43
    ref, A = _prompt_ref(s, [1], [2700])
    _check(kernels.attn_prompt(**s), ref, A, BF, False)
    s = _batch(65, HF, 7, 1, D, 64, [20], prefix=2701)
    s["prefix_table"] = s["prefix_table"][:43].contiguous()
    ref, A = _batch_ref(s, [20], 2701)
    _check(kernels.attn_shared(**s), ref, A, HF, False)


@pytest.mark.parametrize("scale", [1e-20, 1e-38, 1e-40, 1e-45])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (BF, 256)])
def test_a_scale_next_to_zero_gives_the_mean(scale, dtype, D):
    lens = [3000, 200, 0]
    for prefix in (None, 1500):
        s = dict(_batch(66, dtype, 8, 2, D, 64, lens, prefix=prefix), scale=scale)
        ref, A = _batch_ref(s, lens, prefix or 0)
        _check((kernels.attn_shared if prefix else kernels.attn_batch)(**s), ref, A, dtype, not prefix)
    s = _prompt(67, dtype, 8, 2, D, 64, [5, 70], [3000, 3], scale=scale)
    ref, A = _prompt_ref(s, [5, 70], [3000, 3])
    _check(kernels.attn_prompt(**s), ref, A, dtype, False)


def _odd_ones(x, pitch=4097):
    """x with the strides of its dimensions of size 1 replaced by an odd number."""
    return x.as_strided(x.shape, [pitch if n == 1 else s for n, s in zip(x.shape, x.stride())])


@pytest.mark.parametrize("hq,hk", [(8, 1), (1, 1), (8, 2)])
def test_odd_strides_of_dimensions_of_size_one(hq, hk):
    """One token, one head, one page: strides that no address is formed with, as torch leaves them after a cut."""
    g = _gen(68)
    kc, vc = _cache(g, 1, hk, 64, 128, BF)
    q, k, v = _rand(g, 1, hq, 128), _rand(g, 1, hk, 128), _rand(g, 1, hk, 128)
    cos, sin = _rope(g, 64, 128, BF, False, False)
    one, zero = _i32([30]), _i32([[0]])
    caches = [[c.clone() for c in (kc, vc)] for _ in range(2)]
    res = []
    for odd, (a, b) in zip((lambda x: x, _odd_ones), caches):
        q1 = kernels.kv_append(odd(q), odd(k), odd(v), cos, sin, _i32([0, 1]), one, zero, odd(a), b)
        res.append([q1, kernels.attn_prompt(odd(q), a, odd(b), _i32([0, 1]), one, zero, 0.1),
                    kernels.attn_batch(odd(q1), odd(a), b, one, zero, 0.1),
                    kernels.attn_shared(odd(q1), odd(a), odd(b), one, zero, one, zero[0], 0.1), a, b])
    for x, y in zip(*res):
        assert torch.equal(x, y)


def test_no_sequences():
    g = _gen(69)
    kc, vc = _cache(g, 4, 2, 16, 128, BF)
    k0, v0 = kc.clone(), vc.clone()
    cos, sin = _rope(g, 8, 128, BF, False, False)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    for W in (0, 3):
        table = torch.zeros(0, W, dtype=torch.int32, device=DEV)
        q = _rand(g, 0, 8, 128)
        assert kernels.attn_batch(q, kc, vc, none, table, 0.1).shape == (0, 8, 128)
        for pre in (none, _i32([1])):
            assert kernels.attn_shared(q, kc, vc, none, table, _i32([3]), pre, 0.1).shape == (0, 8, 128)
        for T in (0, 5):  # five rows that belong to no sequence
            q, k, out = _rand(g, T, 8, 128), _rand(g, T, 2, 128), torch.full((T, 8, 128), 2.0, dtype=BF, device=DEV)
            assert kernels.kv_append(q, k, k, cos, sin, _i32([0]), none, table, kc, vc, qo=out) is out and (out == 2.0).all()
            assert kernels.attn_prompt(q, kc, vc, _i32([0]), none, table, 0.1, out=out) is out and (out == 2.0).all()
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_tables_without_pages():
    """Sequences of length 0 read nothing; a length past such a table is NaN, as past any."""
    s = _batch(70, BF, 8, 2, 128, 16, [0, 0, 40], prefix=70)
    table = torch.empty(3, 0, dtype=torch.int32, device=DEV)
    none = dict(s, table=table, kv_len=_i32([0, 0, 1]))
    got = kernels.attn_shared(**none)
    want = kernels.attn_shared(**dict(s, kv_len=_i32([0, 0, 0])))
    assert torch.equal(got[:2], want[:2]) and got[2].isnan().all()
    got = kernels.attn_shared(**dict(s, prefix_table=table[0], prefix_len=_i32([0])))
    own = {k: v for k, v in s.items() if not k.startswith("prefix")}
    ref, A = _batch_ref(own, [0, 0, 40])
    _check(got, ref, A, BF, False)
    assert kernels.attn_shared(**dict(s, prefix_table=table[0])).isnan().all()
    got = kernels.attn_batch(**dict(own, table=table, kv_len=_i32([0, 5, -1])))
    assert (got[0] == 0).all() and got[1].isnan().all() and (got[2] == 0).all()
    q, k = _rand(_gen(71), 2, 8, 128), _rand(_gen(72), 2, 2, 128)
    cos, sin = _rope(None, 8, 128, BF, False, False)
    k0 = s["kc"].clone()
    assert kernels.kv_append(q, k, k, cos, sin, _i32([0, 2, 2, 2]), _i32([2, 0, 0]), table, s["kc"], s["vc"]).isnan().all()
    assert torch.equal(s["kc"], k0)
    got = kernels.attn_prompt(q, s["kc"], s["vc"], _i32([0, 2, 2, 2]), _i32([0, 0, 0]), table, 0.1)  # positions -2 and -1
    assert (got == 0).all()
