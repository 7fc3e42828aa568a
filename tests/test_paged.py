"""The paged K/V cache's entry points on the CPU: what they refuse, before anything reaches the device."""

import ctypes
import os
import re
import shutil
import subprocess
import tempfile

import pytest
import torch

from wisp import _lib, kernels

FAKE = 0x100000  # never dereferenced: every call below ends at a check
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

CACHE = dict(kc=FAKE, vc=FAKE, pages=8, page=16, page_stride=8 * 16 * 128, head_stride=16 * 128, row_stride=128)


def _append(**kw):
    a = dict(q=FAKE, q_ts=4096, q_hs=128, k=FAKE, k_ts=512, k_hs=128, v=FAKE, v_ts=512, v_hs=128, qw=FAKE, kw=FAKE, eps=1e-6,
             cos=FAKE, sin=FAKE, cs_rows=100, rot=128, cs_dtype=0, inter=0, cu=FAKE, kv_len=FAKE, table=FAKE, width=4, B=2,
             T=5, hq=32, hk=4, d=128, dtype=0, **CACHE, qo=FAKE, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.lib().wisp_kv_append(*a.values())


def _prompt(**kw):
    a = dict(q=FAKE, q_ts=4096, q_hs=128, **CACHE, cu=FAKE, kv_len=FAKE, table=FAKE, width=4, B=2, T=5, hq=32, hk=4, d=128,
             dtype=0, scale=0.1, ws=FAKE, out=FAKE, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.lib().wisp_attn_prompt(*a.values())


def _batch(**kw):
    a = dict(q=FAKE, q_ts=4096, q_hs=128, **CACHE, kv_len=FAKE, table=FAKE, width=4, prefix_len=FAKE, prefix_table=FAKE,
             prefix_width=2, B=2, hq=32, hk=4, d=128, dtype=0, scale=0.1, ws=FAKE, out=FAKE, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _lib.lib().wisp_attn_batch(*a.values())


BOTH = [
    (dict(dtype=2), b"dtype"), (dict(d=96), b"head dim"), (dict(d=512), b"head dim"), (dict(hq=30), b"multiple of hk"),
    (dict(hk=0), b"multiple of hk"), (dict(hq=2048, hk=4), b"at most 1024"), (dict(page=8), b"page"), (dict(page=48), b"page"),
    (dict(pages=0), b"at least one page"), (dict(B=0), b"B must"), (dict(width=0), b"table"), (dict(width=1 << 28), b"table"),
    (dict(kc=None), b"null cache"), (dict(row_stride=64), b"strides"), (dict(head_stride=-128), b"strides"),
    (dict(row_stride=1 << 23), b"row stride"),
]


@pytest.mark.parametrize("call", [_append, _prompt, _batch])
@pytest.mark.parametrize("args,needle", BOTH)
def test_cache_arguments(call, args, needle):
    assert call(**args) == _lib.WISP_EINVAL
    assert needle in _lib.lib().wisp_last_error(), _lib.lib().wisp_last_error()


@pytest.mark.parametrize("call", [_append, _prompt, _batch])
@pytest.mark.parametrize("args", [dict(kc=FAKE + 8), dict(vc=FAKE + 2), dict(page_stride=16385), dict(head_stride=2052),
                                  dict(row_stride=132), dict(q=FAKE + 4), dict(q_ts=4100), dict(q_hs=130)])
def test_cache_alignment(call, args):
    assert call(**args) == _lib.WISP_EALIGN


@pytest.mark.parametrize("call,args,needle", [
    (_append, dict(T=-1), b"T must"), (_append, dict(rot=8), b"rot"), (_append, dict(rot=136), b"rot"),
    (_append, dict(rot=72), b"rot"), (_append, dict(cs_rows=0), b"row"), (_append, dict(cs_dtype=1), b"cos and sin"),
    (_append, dict(qw=None), b"both or neither"), (_append, dict(qo=None), b"null"), (_append, dict(table=None), b"null"),
    (_prompt, dict(T=-1), b"T * hq"), (_prompt, dict(T=1 << 26), b"T * hq"), (_prompt, dict(scale=0.0), b"scale"),
    (_prompt, dict(scale=-1.0), b"scale"), (_prompt, dict(scale=float("inf")), b"scale"),
    (_prompt, dict(scale=float("nan")), b"scale"), (_prompt, dict(out=None), b"null"), (_prompt, dict(cu=None), b"null"),
    (_prompt, dict(ws=None, width=400), b"workspace"),
    (_batch, dict(scale=0.0), b"scale"), (_batch, dict(ws=None), b"workspace"),
    (_batch, dict(ws=None, prefix_width=0, width=400), b"workspace"), (_batch, dict(prefix_len=None), b"null"),
    (_batch, dict(prefix_width=-1), b"prefix"), (_batch, dict(prefix_width=1 << 28), b"prefix"),
    (_batch, dict(kv_len=None), b"null"),
])
def test_own_arguments(call, args, needle):
    assert call(**args) == _lib.WISP_EINVAL
    assert needle in _lib.lib().wisp_last_error(), _lib.lib().wisp_last_error()


def test_other_alignment():
    for call, args in ((_append, dict(cos=FAKE + 4)), (_append, dict(k=FAKE + 8)), (_append, dict(qo=FAKE + 8)),
                       (_append, dict(v_hs=4)), (_append, dict(kw=FAKE + 2)), (_prompt, dict(out=FAKE + 8)),
                       (_batch, dict(out=FAKE + 8)), (_batch, dict(ws=FAKE + 8))):
        assert call(**args) == _lib.WISP_EALIGN, args


def test_no_tokens_is_a_call_that_does_nothing():
    assert _append(T=0) == _lib.WISP_OK and _prompt(T=0) == _lib.WISP_OK
    assert _append(T=0, q=None, qo=None) == _lib.WISP_OK  # torch's empty tensors have no address


def test_workspaces():
    L = _lib.lib()
    assert L.wisp_attn_prompt_ws_bytes(16384, 1, 32, 4, 128, 64, 256) == 0  # tiles enough for every CU
    assert L.wisp_attn_prompt_ws_bytes(0, 1, 32, 4, 128, 64, 256) == 0
    assert L.wisp_attn_prompt_ws_bytes(8, 1, 32, 4, 128, 64, 256) > 0
    assert L.wisp_attn_prompt_ws_bytes(8, 1, 30, 4, 128, 64, 256) == -1
    assert L.wisp_attn_batch_ws_bytes(0, 32, 4, 128, 64, 99, 0) == -1
    assert L.wisp_attn_batch_ws_bytes(8, 32, 4, 128, 64, 0, 0) == -1
    assert L.wisp_attn_batch_ws_bytes(8, 32, 4, 128, 64, 2, 0) == 0  # short tables: no pieces, no records
    own = L.wisp_attn_batch_ws_bytes(8, 32, 4, 128, 64, 99, 0)
    assert 0 < own < L.wisp_attn_batch_ws_bytes(8, 32, 4, 128, 64, 99, 256)


def test_cpu_tensors_and_wrong_types_are_refused():
    bf = torch.bfloat16
    q, k = torch.zeros(3, 8, 64, dtype=bf), torch.zeros(3, 2, 64, dtype=bf)
    kc = torch.zeros(4, 2, 16, 64, dtype=bf)
    cs = torch.zeros(9, 64, dtype=bf)
    cu, n, t = (torch.zeros(s, dtype=torch.int32) for s in ((3,), (2,), (2, 2)))
    calls = {
        "append": lambda **x: kernels.kv_append(**dict(dict(q=q, k=k, v=k, cos=cs, sin=cs, cu=cu, kv_len=n, table=t, kc=kc, vc=kc), **x)),
        "prompt": lambda **x: kernels.attn_prompt(**dict(dict(q=q, kc=kc, vc=kc, cu=cu, kv_len=n, table=t, scale=1.0), **x)),
        "batch": lambda **x: kernels.attn_batch(**dict(dict(q=q[:2], kc=kc, vc=kc, kv_len=n, table=t, scale=1.0), **x)),
        "shared": lambda **x: kernels.attn_shared(**dict(dict(q=q[:2], kc=kc, vc=kc, kv_len=n, table=t, scale=1.0,
                                                              prefix_len=n[:1], prefix_table=n), **x)),
    }
    for call in calls.values():
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
        with pytest.raises(TypeError):
            call(q=q.float()[: 2 if call in (calls["batch"], calls["shared"]) else 3])
        with pytest.raises(TypeError):
            call(kc=kc.half())
        with pytest.raises(TypeError):
            call(table=t.long())
        with pytest.raises(AssertionError):
            call(vc=kc[:2])
        with pytest.raises(AssertionError):
            call(kc=torch.zeros(4, 3, 16, 64, dtype=bf), vc=torch.zeros(4, 3, 16, 64, dtype=bf))
        with pytest.raises(AssertionError):
            call(kc=kc.transpose(2, 3).contiguous().transpose(2, 3), vc=kc.transpose(2, 3).contiguous().transpose(2, 3))


@pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="hipcc not installed")
def test_m0_is_written_by_the_direct_loads_only():
    """csrc/paged_attn.hip writes M0 in inline assembly, a register the compiler treats as reserved (the clobber is advisory):
    no instruction outside those statements may read or write it."""
    with tempfile.TemporaryDirectory() as d:
        out = os.path.join(d, "k.s")
        cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-mcode-object-version=5", "-Xclang",
               "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", "-o", out,
               os.path.join(ROOT, "wisp-runtime_amd", "csrc", "paged_attn.hip")]
        r = subprocess.run(cmd, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-2000:]
        asm = open(out).read()
    inside, dma, other = False, 0, []
    for line in asm.splitlines():
        s = line.strip()
        if s.startswith(";;#ASMSTART"):
            inside = True
        elif s.startswith(";;#ASMEND"):
            inside = False
        elif inside:
            dma += "global_load_lds_dwordx4" in s
        elif re.search(r"\bm0\b", s.split(";", 1)[0]):
            other.append(s)
    assert dma > 0 and not other, other[:5]


def test_token_counts_past_any_call_are_refused():
    L = _lib.lib()
    for T in (1 << 31, 1 << 62):
        assert L.wisp_attn_prompt_ws_bytes(T, 1, 32, 4, 128, 64, 256) == -1
        assert _prompt(T=T) == -1
        assert _append(T=T) == -1


def test_workspaces_keep_records_aligned():
    """7 heads and 21 parts (43 tiles of 64 positions): an odd number of records, whose sums begin at a multiple of 16 bytes."""
    L = _lib.lib()
    recs = 7 * 21
    assert L.wisp_attn_prompt_ws_bytes(1, 1, 7, 1, 64, 64, 43) == recs * 8 + 8 + recs * 64 * 4
    assert L.wisp_attn_batch_ws_bytes(1, 7, 1, 64, 64, 1, 43) == recs * 8 + 8 + recs * 64 * 4
    assert L.wisp_attn_prompt_ws_bytes(2, 1, 7, 1, 64, 64, 43) == 2 * recs * 8 + 2 * recs * 64 * 4


def test_workspace_alignment():
    for call in (_prompt, _batch):
        for by in (4, 8):
            assert call(ws=FAKE + by) == _lib.WISP_EALIGN
            assert b"ws" in _lib.lib().wisp_last_error()


@pytest.mark.parametrize("call", [_prompt, _batch])
def test_a_scale_past_the_exponent_is_refused(call):
    assert call(scale=3e38) == _lib.WISP_EINVAL  # times log2(e): infinite
    assert b"scale" in _lib.lib().wisp_last_error()


def test_strides_of_dimensions_of_size_one_say_nothing():
    bf = torch.bfloat16
    x = torch.zeros(40000, dtype=bf)
    for t, want in ((x.as_strided((1, 8, 128), (4097, 128, 1)), 128), (x.as_strided((1, 8, 128), (4097, 136, 1)), 136)):
        y, at, ts, hs = kernels._rows(t, "q")
        assert at == t.data_ptr() and ts % 8 == 0 and hs == want  # as it is
    y, at, ts, hs = kernels._rows(x.as_strided((5, 1, 128), (136, 3, 1)), "q")
    assert at == x.data_ptr() and ts == 136 and hs % 8 == 0
    y, at, ts, hs = kernels._rows(x.as_strided((1, 8, 128), (4097, 132, 1)), "q")
    assert at != x.data_ptr() and (ts, hs) == (1024, 128)  # a copy
    y, at, ts, hs = kernels._rows(x[4:].as_strided((1, 8, 128), (4097, 128, 1), 4), "q")
    assert at % 16 == 0 and at != x.data_ptr() + 8 and (ts, hs) == (1024, 128)
    q, table = torch.zeros(1, 8, 128, dtype=bf), torch.zeros(1, 1, dtype=torch.int32)
    one_page = x.as_strided((1, 2, 64, 128), (16385, 8192, 128, 1)), x.as_strided((1, 2, 64, 128), (7, 8192, 128, 1))
    assert kernels._paged_cache(q, *one_page, table, "t")[4][4:] == (0, 8192, 128)
    one_head = x.as_strided((3, 1, 64, 128), (8192, 3, 128, 1)), x.as_strided((3, 1, 64, 128), (8192, 8192, 128, 1))
    assert kernels._paged_cache(q, *one_head, table, "t")[4][4:] == (8192, 0, 128)
    with pytest.raises(AssertionError):
        kernels._paged_cache(q, one_head[0], x.as_strided((3, 1, 64, 128), (8704, 8192, 136, 1)), table, "t")


def test_a_cache_without_heads_is_refused():
    kc = torch.zeros(4, 0, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="K/V heads"):
        kernels.attn_batch(torch.zeros(2, 8, 64, dtype=torch.bfloat16), kc, kc, torch.zeros(2, dtype=torch.int32),
                           torch.zeros(2, 1, dtype=torch.int32), 0.1)
