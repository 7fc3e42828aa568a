"""GraphDecoder.prefill(fused=True): the decoder's prompts through kv_append and attn_prompt, on the small Qwen3-MoE of
test_graphdec_gpu.py, with that file's bar against transformers in float32 (the bf16 roundings of three layers)."""

from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

pytest.importorskip("transformers")
from test_graphdec_gpu import _close, _models  # noqa: E402

from wisp.graphdec import GraphDecoder  # noqa: E402


def test_fused_prefill_then_decode_matches_transformers():
    cfg, ref, gpu, rt = _models()
    ids = torch.randint(0, 128, (1, 9), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        out = ref(input_ids=ids, use_cache=True)
        pk = out.past_key_values
        dec = GraphDecoder(gpu, rt, tmax=128)
        lg = dec.prefill(ids[0].cuda(), 0, chunk=4, fused=True)
        err, ok = _close(lg, out.logits[:, -1], 2e-2)
        assert ok, err
        t = out.logits[:, -1].argmax(-1)
        for step in range(6):
            r = ref(input_ids=t[:, None], past_key_values=pk, use_cache=True)
            pk = r.past_key_values
            err, ok = _close(dec.next(t.cuda()), r.logits[:, -1], 2e-2)
            assert ok, (step, err)
            t = r.logits[:, -1].argmax(-1)
    rt.cache.free()


@pytest.mark.parametrize("chunk", [1024, 37, 1])
def test_fused_prefill_stores_what_the_modules_store(chunk):
    """Layer 0's keys differ from the modules' by their two more roundings of u = 2^-8 (after the norm, after the weight: of
    a value and of its partner, 2 u S with S = |k cos| + |k' sin| <= 2 max |k|) and one last one; its values not at all;
    positions past the prompt not at all."""
    cfg, ref, gpu, rt = _models(seed=5, nslots=24)
    ids = torch.randint(0, 128, (70,), generator=torch.Generator().manual_seed(6)).cuda()
    kv = []
    for fused in (False, True):
        dec = GraphDecoder(gpu, rt, tmax=128)
        with torch.no_grad():
            dec.prefill(ids, 0, chunk=chunk, fused=fused)
        assert dec.pos == 70
        kv.append(dec.kv.clone())
    a, b = kv[0].double(), kv[1].double()
    assert torch.equal(kv[0][0, 1], kv[1][0, 1])
    u = 2.0**-8
    top = a[0, 0].abs().amax(-1, keepdim=True)
    assert ((a[0, 0] - b[0, 0]).abs() <= 2 * u * a[0, 0].abs() + 4 * u * top).all()
    assert (kv[1][:, :, :, 70:] == 0).all()
    rt.cache.free()


def test_turns_of_fused_and_plain_prefill_share_the_cache():
    """A prompt whose first turn is prefilled by the modules and whose second, fused, attends it."""
    cfg, ref, gpu, rt = _models(seed=5)
    ids = torch.randint(0, 128, (1, 20), generator=torch.Generator().manual_seed(6))
    with torch.no_grad():
        want = ref(input_ids=ids).logits[:, -1]
        dec = GraphDecoder(gpu, rt, tmax=64)
        dec.prefill(ids[0, :12].cuda(), 0, chunk=5)
        err, ok = _close(dec.prefill(ids[0, 12:].cuda(), 12, chunk=3, fused=True), want, 2e-2)
    assert ok, err
    rt.cache.free()


@pytest.mark.parametrize("turns", [[1500], [700, 1, 640]])
def test_fused_attention_at_length(turns):
    """Layer 0's attention over the static cache, 32 query and 4 K/V heads of 128, in one piece and in turns: against 64 bits
    over the keys and values that it stored, with the bound of test_paged_gpu.py."""
    from test_paged_gpu import _attend, _check, _i32

    from wisp import kernels

    Hq, Hk, D, hid, T = 32, 4, 128, 256, sum(turns)
    g = torch.Generator(device="cuda").manual_seed(7)
    rand = lambda *s: (torch.randn(s, generator=g, device="cuda") * hid**-0.5).to(torch.bfloat16)
    lin = [torch.nn.Linear(hid, h * D, bias=False, device="cuda", dtype=torch.bfloat16) for h in (Hq, Hk, Hk)]
    with torch.no_grad():
        for m in lin:
            m.weight.copy_(rand(*m.weight.shape))
    at = SimpleNamespace(q_proj=lin[0], k_proj=lin[1], v_proj=lin[2])
    w = dict(qn=rand(D) + 1, kn=rand(D) + 1, epsq=1e-6, scale=D**-0.5)
    cap = -(-T // 64) * 64 + 64
    ang = torch.rand(cap, D // 2, generator=g, device="cuda").repeat(1, 2)
    dec = SimpleNamespace(shape=SimpleNamespace(per_layer=[w]), D=D, Hq=Hq, Hk=Hk, cos=ang.cos().to(torch.bfloat16),
                          sin=ang.sin().to(torch.bfloat16), kv=torch.zeros(1, 2, Hk, cap, D, dtype=torch.bfloat16, device="cuda"))
    x = rand(1, T, hid) * hid**0.5
    table, done, got, qs = torch.arange(cap // 64, dtype=torch.int32, device="cuda")[None], 0, [], []
    with torch.no_grad():
        for n in turns:
            xn, cu, kv_len = x[:, done : done + n], _i32([0, n]), _i32([done + n])
            got.append(GraphDecoder._attend_fused(dec, 0, at, xn, cu, kv_len, table).view(n, Hq, D))
            q, k, v = (m(xn).view(n, -1, D) for m in lin)
            other = [torch.zeros(cap // 64, Hk, 64, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
            qs.append(kernels.kv_append(q, k, v, dec.cos, dec.sin, cu, kv_len, table, *other, w["qn"], w["kn"], 1e-6))
            stored = [c.transpose(0, 1).reshape(Hk, cap, D)[:, done : done + n] for c in other]
            for j in range(2):
                assert torch.equal(dec.kv[0, j, :, done : done + n], stored[j])
            done += n
    assert (dec.kv[0, :, :, T:] == 0).all()
    rows = sorted({0, 1, 63, 64, 255, 256, 699, 700, 701, T // 2, T - 2, T - 1})
    kk, vv = dec.kv[0, 0, :, :T].double(), dec.kv[0, 1, :, :T].double()
    ref, A = _attend(torch.cat(qs)[rows], kk, vv, w["scale"], rows)
    _check(torch.cat(got)[rows], ref, A, torch.bfloat16, False)
