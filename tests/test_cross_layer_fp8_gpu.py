"""A cross-attention layer as a model holds it: e4m3 to_q, fused e4m3 to_k | to_v over the encoder's states, cross attention over prompts of
different lengths, e4m3 to_out, and its gradients -- against the same layer in 64 bits without any quantisation.

Bar: an e4m3 rounding is off by at most 2^-4 of the value and uniform within its step: rms 2^-4 / sqrt(3) * sqrt(E[1 / m^2]) over mantissas m
uniform in [1, 2) (E = 1/2) = 0.0255.  Both operands of a product are rounded, and its terms' errors add like independent ones: an e4m3 Linear of
random operands is off by 0.0255 sqrt(2) = 0.036 of its L2 norm.  (The 16-bit roundings, at most 2^-8, are a tenth of that.)
 * o2 = to_out(attention(to_q, to_k, to_v)): the attention passes v's error on (0.036), turns the errors of q and of k into errors of the scores
   (relative to the scores' spread, which is kept at 1 here: a probability moves by as much, 0.036 each), to_out adds its own: at most
   4 * 0.036 = 0.15 if none of them cancels.
 * a gradient adds the products of the backward pass on its way: gx of to_out (0.036), the probabilities' error in both factors of p (dp - D)
   (0.036 * 2 twice, and v's), the last Linear's own (0.036): at most 8 * 0.036 = 0.29.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    import tfmq_dm_amd.ops as ops
    return ops


class Layer:
    """The layer on the kernels: forward keeps what its gradients need."""

    def __init__(self, ops, wq, wk, wv, wo, bo, heads, kv_heads):
        self.ops, self.H, self.G = ops, heads, kv_heads
        self.q, self.kv, self.o = ops.pack_w_fp8(wq.to(DEV)), ops.pack_w_fp8(torch.cat([wk, wv]).to(DEV)), ops.pack_w_fp8(wo.to(DEV), bo.to(DEV))
        self.scale = (wq.shape[0] // heads) ** -0.5

    def forward(self, x, ctx, mask):
        q, kv = self.ops.linear_fp8(x, self.q), self.ops.linear_fp8(ctx, self.kv)
        C = kv.shape[-1] // 2
        o, lse = self.ops.cross_attention(q, kv[..., :C], kv[..., C:], self.H, self.scale, self.G, mask=mask, want_lse=True)
        self.saved = x, ctx, mask, q, kv, o, lse
        return self.ops.linear_fp8(o, self.o)

    def backward(self, gy):
        x, ctx, mask, q, kv, o, lse = self.saved
        C = kv.shape[-1] // 2
        go, gwo = self.ops.linear_fp8_bwd(o, gy, self.o)
        dq, dk, dv = self.ops.cross_attention_bwd(q, kv[..., :C], kv[..., C:], o, lse, go, self.H, self.scale, self.G, mask=mask)
        gx, gwq = self.ops.linear_fp8_bwd(x, dq, self.q)
        gc, gwkv = self.ops.linear_fp8_bwd(ctx, torch.cat([dk, dv], -1), self.kv)
        return dict(x=gx, ctx=gc, wq=gwq, wk=gwkv[:C], wv=gwkv[C:], wo=gwo)


def reference(x, ctx, wq, wk, wv, wo, bo, H, G, mask, gy):
    ls = [t.double().requires_grad_() for t in (x, ctx, wq, wk, wv, wo)]
    x, ctx, wq, wk, wv, wo = ls
    B, T, _ = x.shape
    L = ctx.shape[1]
    d = wq.shape[0] // H
    q = (x @ wq.t()).view(B, T, H, d).transpose(1, 2)
    k = (ctx @ wk.t()).view(B, L, G, d).transpose(1, 2).repeat_interleave(H // G, 1)
    v = (ctx @ wv.t()).view(B, L, G, d).transpose(1, 2).repeat_interleave(H // G, 1)
    s = (q @ k.transpose(-1, -2) * d ** -0.5).masked_fill(~mask[:, None, None], -1e300)
    p = s.softmax(-1) * mask[:, None, None]
    y = (p @ v).transpose(1, 2).reshape(B, T, H * d) @ wo.t() + bo.double()
    y.backward(gy.double())
    return y.detach(), dict(zip(("x", "ctx", "wq", "wk", "wv", "wo"), (t.grad for t in ls)))


def rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm())


def make(B, T, L, D, H, G, d, dt, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    C, Dc = H * d, D + 24
    w = (r(C, D) * D ** -0.5, r(G * d, Dc) * Dc ** -0.5, r(G * d, Dc) * Dc ** -0.5, r(D, C) * C ** -0.5, r(D))
    mask = torch.rand(B, L, generator=g) < 0.8
    mask[:, 0] = True
    if B > 1:
        mask[-1] = False            # a prompt of no tokens: its rows of the attention are zero
    return r(B, T, D).to(dt), r(B, L, Dc).to(dt), w, mask, r(B, T, D).to(dt)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,L,D,H,G,d", [(2, 256, 77, 320, 8, 8, 40), (3, 65, 77, 200, 4, 2, 64), (1, 1, 300, 136, 2, 1, 80), (2, 600, 300, 256, 4, 4, 64)])
def test_layer_and_its_gradients(ops, B, T, L, D, H, G, d, dt):
    x, ctx, w, mask, gy = make(B, T, L, D, H, G, d, dt, B + T + L)
    ry, rg = reference(x, ctx, *w, H, G, mask, gy)
    layer = Layer(ops, *w, H, G)
    y = layer.forward(x.to(DEV), ctx.to(DEV), mask.to(DEV))
    assert y.dtype == dt and rel(y, ry) <= 0.15
    if B > 1:       # the row of an empty prompt is the bias alone (rounded once)
        b = w[4].double().expand_as(ry[-1])
        assert bool(((y[-1].double().cpu() - b).abs() <= torch.finfo(dt).eps / 2 * b.abs()).all())
    g = layer.backward(gy.to(DEV))
    for n, ref in rg.items():
        assert g[n].shape == ref.shape and rel(g[n], ref) <= 0.29, (n, rel(g[n], ref))
    if B > 1:
        assert not g["ctx"][-1].any() and not g["x"][-1].any()


def test_layer_in_a_graph_between_eager_runs(ops):
    """Forward and gradients recorded once and replayed over other inputs, with the same layer run eagerly in between."""
    H, G, d, D = 4, 2, 64, 200
    sets = [make(2, 130, 77, D, H, G, d, torch.float16, s) for s in range(4)]
    layer = Layer(ops, *sets[0][2], H, G)

    def step(x, ctx, mask, gy):
        y = layer.forward(x, ctx, mask)
        return [y] + list(layer.backward(gy).values())

    def on(s):
        return [t.to(DEV) for t in (s[0], s[1], s[3], s[4])]
    bufs = on(sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*bufs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*bufs)
    for s in sets[1:] + sets[:1]:
        for b, t in zip(bufs, on(s)):
            b.copy_(t)
        graph.replay()
        eager = step(*on(s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
