"""GraphDecoder.prefill(fused=True): the decoder's prompts through kv_append and attn_prompt, on the small Qwen3-MoE of
test_graphdec_gpu.py, with that file's bar against transformers in float32 (the bf16 roundings of three layers)."""

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
