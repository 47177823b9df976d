"""LdmUNetEngine.forward(context_mask=...) at the full SD v1 size: row chains, fused feed-forward and fused to_k | to_v around the masked attention
(head dims 40, 80 and 160).  The bar against the unmasked run is the one between the fp16 and the fp32 activation stream at this size, 4e-2: the masked
attention rounds its output to fp16 in front of the 8-bit quantizer."""
import pytest
import torch

from test_full_size_properties_gpu import DEV, _engine_of, sd  # noqa: F401  (sd: the module's engine fixture)

pytestmark = pytest.mark.gpu


def test_prompts_of_different_lengths(sd, monkeypatch):  # noqa: F811
    run, fwd, info = sd
    eng = _engine_of(fwd)
    g = torch.Generator().manual_seed(21)
    x = torch.randn(4, 64, 64, 4, generator=g).to(DEV)
    ctx = torch.randn(4, 77, 768, generator=g).to(DEV)
    lens = torch.tensor([77, 9, 32, 1], device=DEV)
    mask = torch.arange(77, device=DEV)[None] < lens[:, None]
    junk = torch.where(mask[..., None], ctx, torch.full_like(ctx, float("nan")))
    with torch.cuda.stream(info["stream"]):
        info["step"].zero_()
        plain = eng.forward(x, None, ctx).clone()
        full = eng.forward(x, None, ctx, context_mask=torch.ones_like(mask)).clone()
        a = eng.forward(x, None, ctx, context_mask=mask).clone()
        b = eng.forward(x, None, junk, context_mask=mask).clone()
        one = eng.forward(x[1:2].contiguous(), None, ctx[1:2, :9].contiguous(), context_mask=mask[1:2, :9]).clone()
        monkeypatch.setenv("TFMQ_FUSED_KV", "0")
        c = eng.forward(x, None, ctx, context_mask=mask).clone()
        monkeypatch.delenv("TFMQ_FUSED_KV")
        monkeypatch.setenv("TFMQ_ROW_CHAIN", "0")
        monkeypatch.setenv("TFMQ_FF_FUSED", "0")
        d = eng.forward(x, None, ctx, context_mask=mask).clone()
        info["stream"].synchronize()
    assert torch.isfinite(a).all() and torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)
    assert torch.equal(a[1:2], one) and torch.equal(a[0], full[0]) and not torch.equal(a[1:], full[1:])
    assert float((full - plain).norm() / plain.norm()) <= 4e-2
