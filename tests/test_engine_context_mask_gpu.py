"""LdmUNetEngine.forward(context_mask=...): prompts of different lengths in one batch, on the fp16-operand cross attention.

Bars: the masked run rounds the attention output to fp16 before its 8-bit quantizer, the unmasked one quantises the fp32 value, so the two differ
by single bins of that quantizer -- the same change of rounding as between the fp16 and the fp32 activation stream, whose bar is 3e-2."""
import pytest
import torch

from test_engine_ldm_gpu import CFG, DEV, T, layerq, nhwc, rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def run(golden):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tfmq_dm_amd.engine import LayerQ, LdmUNetEngine
    g = golden("f11_ldm_tiny")
    sd = {k[3:]: T(g[k]) for k in g.files if k.startswith("sd/")}
    wq, qtable = layerq(g, LayerQ, True)
    eng = LdmUNetEngine(sd, CFG, DEV)
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    eng.prepare(wq, qtable.repeat(4, 1, 1).contiguous().to(DEV), step)
    x, t, ctx = nhwc(T(g["x"])), T(g["t"]).float().to(DEV), T(g["ctx"]).float().to(DEV)
    return eng, x, t, ctx


def lengths(ctx, *n):
    return torch.arange(ctx.shape[1], device=ctx.device)[None] < torch.tensor(n, device=ctx.device)[:, None]


def test_full_mask_equals_no_mask(run):
    eng, x, t, ctx = run
    a = eng.forward(x, t, ctx)
    b = eng.forward(x, t, ctx, context_mask=lengths(ctx, *[ctx.shape[1]] * ctx.shape[0]))
    assert rel_l2(b, a) <= 3e-2


def test_masked_tokens_are_as_if_absent(run):
    """An item of n real tokens equals its own run on the context of those n alone; what the other tokens hold does not matter."""
    eng, x, t, ctx = run
    B, L = ctx.shape[:2]
    n = [max(1, L - 2 * (i + 1)) for i in range(B)]
    mask = lengths(ctx, *n)
    a = eng.forward(x, t, ctx, context_mask=mask)
    for i in range(B):
        alone = eng.forward(x, t, ctx[:, :n[i]].contiguous(), context_mask=lengths(ctx[:, :n[i]], *[n[i]] * B))
        assert torch.equal(alone[i], a[i]), i
        assert rel_l2(a[i], eng.forward(x, t, ctx[:, :n[i]].contiguous())[i]) <= 3e-2, i
    full = eng.forward(x, t, ctx)
    assert not torch.equal(full, a) and rel_l2(full, a) > 0
    for junk in (7.0, float("inf"), float("nan")):
        other = torch.where(mask[..., None], ctx, torch.full_like(ctx, junk))
        assert torch.equal(eng.forward(x, t, other, context_mask=mask), a), junk


def test_holes_and_an_empty_row(run):
    """A mask with a hole equals the context without that token (attention has no positions); a row that attends to nothing stays finite."""
    eng, x, t, ctx = run
    B, L = ctx.shape[:2]
    keep = [j for j in range(L) if j != 1]
    mask = torch.ones(B, L, dtype=torch.bool, device=DEV)
    mask[:, 1] = False
    a = eng.forward(x, t, ctx, context_mask=mask)
    b = eng.forward(x, t, ctx[:, keep].contiguous(), context_mask=torch.ones(B, L - 1, dtype=torch.bool, device=DEV))
    assert rel_l2(a, b) <= 3e-2
    mask = lengths(ctx, *([0] + [L] * (B - 1)))
    c = eng.forward(x, t, ctx, context_mask=mask)
    assert bool(torch.isfinite(c).all())
    d = eng.forward(x, t, ctx, context_mask=lengths(ctx, *[L] * B))
    assert torch.equal(c[1:], d[1:]) and not torch.equal(c[0], d[0])


def test_guidance_pair_and_one_token(run):
    eng, x, t, ctx = run
    B, L = ctx.shape[:2]
    c2 = torch.cat([ctx.flip(1), ctx])
    m2 = lengths(c2, *([1] * B + [L - 1] * B))
    t2 = t[:1].repeat(2 * B)
    full = eng.forward(torch.cat([x, x]), t2, c2, context_mask=m2)
    assert torch.equal(eng.forward(x, t2, c2, pair_prefix=True, context_mask=m2), full)
    one = c2[:, :1].contiguous()
    masked = eng.forward(torch.cat([x, x]), t2, one, context_mask=torch.ones(2 * B, 1, dtype=torch.bool, device=DEV))
    assert rel_l2(masked, eng.forward(torch.cat([x, x]), t2, one)) <= 3e-2


def test_replayed_graph_reads_the_mask(run):
    eng, x, t, ctx = run
    B, L = ctx.shape[:2]
    mask = lengths(ctx, *[L] * B)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            eng.forward(x, t, ctx, context_mask=mask)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = eng.forward(x, t, ctx, context_mask=mask)
    for n in (L, 2, L - 1):
        m = lengths(ctx, *[n] * B)
        mask.copy_(m)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eng.forward(x, t, ctx, context_mask=m)), n


def test_refusals(run, golden):
    from tfmq_dm_amd._lib import TfmqError
    from tfmq_dm_amd.engine import LdmUNetEngine
    eng, x, t, ctx = run
    B, L = ctx.shape[:2]
    ok = torch.ones(B, L, dtype=torch.bool, device=DEV)
    for bad in (ok.float(), ok[:, :-1], ok[:-1], ok.cpu()):
        with pytest.raises(TfmqError, match="context_mask"):
            eng.forward(x, t, ctx, context_mask=bad)
    with pytest.raises(TfmqError, match="context_mask"):
        eng.forward(x, t, ctx, context_mask=ok, taps={})
    g = golden("f11_ldm_tiny")
    fp = LdmUNetEngine({k[3:]: T(g[k]) for k in g.files if k.startswith("sd/")}, CFG, DEV)
    fp.prepare()
    with pytest.raises(TfmqError, match="context_mask"):
        fp.forward(x, t, ctx, context_mask=ok)


@pytest.mark.parametrize("kind", ["GraphLatentDdimSampler", "GraphLatentPlmsSampler"])
@pytest.mark.parametrize("pair", ["0", "1"])
def test_captured_samplers_take_masks(run, kind, pair, monkeypatch):
    """Samples of prompts of three tokens, padded to five and masked, equal the samples of the three alone; the masks change between runs of one
    captured sampler; without masks every token counts."""
    from tfmq_dm_amd._lib import TfmqError
    from tfmq_dm_amd.ldm import sampler as S
    monkeypatch.setenv("TFMQ_PAIR_PREFIX", pair)
    eng, x, t, ctx = run
    B, L = ctx.shape[:2]
    cls, n = getattr(S, kind), L - 2
    uc = ctx.flip(0) * 0.5
    xT = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).to(DEV)
    ac = S.alphas_cumprod_linear()

    def sample(smp, *a, **k):
        out = smp.sample_nhwc(xT, *a, **k)
        smp.stream.synchronize()
        return out.clone()
    padded = cls(eng, 4, B, (4, 8, 8), (L, ctx.shape[2]), scale=7.5, alphas_cumprod=ac, context_masks=True).capture()
    junk = lambda c: torch.cat([c[:, :n], torch.full_like(c[:, n:], 9.0)], 1)      # noqa: E731
    m = lengths(ctx, *[n] * B)
    every = sample(padded, ctx, uc)
    a = sample(padded, junk(ctx), junk(uc), cond_mask=m, uncond_mask=m)
    assert torch.equal(sample(padded, ctx, uc), every) and not torch.equal(a, every)
    short = cls(eng, 4, B, (4, 8, 8), (n, ctx.shape[2]), scale=7.5, alphas_cumprod=ac, context_masks=True).capture()
    assert torch.equal(sample(short, ctx[:, :n], uc[:, :n]), a)
    for bad in (m.float(), m[:, :-1]):
        with pytest.raises(TfmqError, match="mask"):
            padded.sample_nhwc(xT, ctx, uc, cond_mask=bad)
    plain = cls(eng, 4, B, (4, 8, 8), (L, ctx.shape[2]), scale=7.5, alphas_cumprod=ac)
    with pytest.raises(TfmqError, match="context_masks"):
        plain.sample_nhwc(xT, ctx, uc, cond_mask=m)
    assert rel_l2(every, sample(plain, ctx, uc)) <= 8e-2      # (the bar of a guided four-step trajectory: guidance amplifies a step's 3e-2)


def test_a_refused_forward_leaves_no_mask_behind(run, golden):
    """A forward that raises inside a block (here: a layer that is not quantised cannot take a mask) ends like any other: a block run on its own afterwards
    takes no mask."""
    from tfmq_dm_amd._lib import TfmqError
    from tfmq_dm_amd.engine import LdmUNetEngine
    eng, x, t, ctx = run
    g = golden("f11_ldm_tiny")
    fp = LdmUNetEngine({k[3:]: T(g[k]) for k in g.files if k.startswith("sd/")}, CFG, DEV)
    fp.prepare()
    name = next(n[:-len(".attn2.to_q")] for n in fp.layers if n.endswith(".attn2.to_q"))
    C = fp.sd[name + ".norm2.weight"].shape[0]
    tok = torch.randn(ctx.shape[0], 16, C, generator=torch.Generator().manual_seed(1)).to(DEV)
    fp.forward(x, t, ctx)          # (the stream's type is that of the last forward)
    fp._ctx_pad = None
    want = fp._tblock(name, tok, ctx)
    with pytest.raises(TfmqError, match="context_mask"):
        fp.forward(x, t, ctx, context_mask=lengths(ctx, *[1] * ctx.shape[0]))
    fp._ctx_pad = None
    assert torch.equal(fp._tblock(name, tok, ctx), want)
