"""K17: the e4m3 Linear with one fp32 scale per block of 128 (ops.quantize_fp8 / pack_w_fp8 / linear_fp8 / linear_fp8_bwd) against a 64-bit
oracle of the definition.  Bytes and scales are compared exactly.  A product's bound counts its roundings: with A = sum |x^| |w^| over the row,
 * the 128 products of a block are summed in fp32, 128 additions of at most 2^-23 each (twice half a step: the unit may truncate);
   for 16-bit outputs the 8-bit matrix instruction aligns every 8 products to their largest and truncates below 2^-13 of it: the seven others
   lose less than 2^-13 of the largest each, so at most 7 2^-13 max|x^| max|w^| per group of 8 channels,
 * one fp32 rounding for the scale product, one for each block's FMA and one for the bias: (Kb + 2) 2^-24,
 * the rounding to the output type: half a step of it, eps / 2 of the value.
"""
import pytest
import torch

import _fp8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    import tfmq_dm_amd.ops as ops
    return ops


def _x(M, K, dt, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + M * 31 + K)
    x = torch.randn(M, K, generator=g) * (1 + 7 * (torch.rand(K, generator=g) < 0.05).float())
    return x.to(dt)


def _bytes(q):
    return q.cpu().view(torch.float8_e4m3fn).double()


def _group_max(q):
    """[R, K] -> [R, ceil(K / 8)]: the largest magnitude of every 8 channels."""
    R, K = q.shape
    return torch.nn.functional.pad(q.abs(), (0, -K % 8)).view(R, -1, 8).amax(-1)


def _terms(x, w):
    """sum |x^| |w^| and the sum over groups of 8 channels of the product of their largest magnitudes."""
    return x.abs() @ w.abs().t(), _group_max(x) @ _group_max(w).t()


def _bound(A, ref, Kb, dt):
    A, G = A
    acc = (128 * 2.0 ** -23 + (Kb + 2) * 2.0 ** -24) * A + (0 if dt == torch.float32 else 7 * 2.0 ** -13 * G)
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0          # half a step of fp16's subnormals
    return acc + (0 if dt == torch.float32 else torch.finfo(dt).eps / 2) * (ref.abs() + acc) + tiny


def _check(y, ref, A, Kb, dt):
    y = y.double().cpu()
    assert y.shape == ref.shape
    bad = (y - ref).abs() > _bound(A, ref, Kb, dt)
    assert not bad.any(), (int(bad.sum()), float(((y - ref).abs() / _bound(A, ref, Kb, dt)).max()))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (17, 128), (16, 129), (77, 320), (33, 1000)])
def test_quantize_rows_is_the_definition(ops, M, K, dt):
    x = _x(M, K, dt)
    x[0] = 0                                                   # a block of zeros
    if M > 2:
        x[1] *= 2.0 ** -12                                     # fp16 subnormals among them
    f = ops.quantize_fp8(x.to(DEV))
    q, s = O.quant_rows(x)
    Kb = (K + 127) // 128
    assert f.q.shape == (M, Kb * 128) and f.scale.shape == (Kb, M)
    assert torch.equal(_bytes(f.q)[:, :K], q) and (f.q[:, K:] == 0).all()
    assert torch.equal(f.scale.cpu().double(), s.t())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (5, 64), (128, 65), (300, 130)])
def test_quantize_columns_is_the_definition(ops, M, K, dt):
    x = _x(M, K, dt)
    q, s = ops._quant_cols_fp8(x.to(DEV), "test")
    qr, sr = O.quant_rows(x.t().contiguous())
    assert torch.equal(_bytes(q)[:, :M], qr) and (q[:, M:] == 0).all()
    assert torch.equal(s.cpu().double(), sr.t())


@pytest.mark.parametrize("N,K", [(1, 1), (31, 7), (128, 128), (129, 320), (333, 257)])
def test_pack_weight_is_the_definition(ops, N, K):
    w = _x(N, K, torch.float32, 3)
    pw = ops.pack_w_fp8(w.to(DEV))
    q, s = O.quant(w, 128)
    assert torch.equal(_bytes(pw.q)[:, :K], q) and (pw.q[:, K:] == 0).all()
    assert torch.equal(_bytes(pw.qt)[:, :N], q.t()) and (pw.qt[:, N:] == 0).all()
    assert torch.equal(pw.scale.cpu().double(), s[::128])
    # a checkpoint in this form: the same layout
    ld = ops.load_w_fp8(pw.q.view(torch.float8_e4m3fn)[:, :K].contiguous(), pw.scale)
    assert torch.equal(ld.q, pw.q) and torch.equal(ld.qt, pw.qt) and torch.equal(ld.scale, pw.scale)


# one row, both sides of the one-launch form's limit and of the tile edges, ragged K and N
SHAPES = [(1, 1, 1), (1, 1280, 320), (2, 7, 33), (32, 129, 130), (33, 128, 128), (77, 768, 320), (128, 320, 127), (129, 520, 333), (300, 64, 1),
          (513, 1280, 640)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_vs_float64(ops, M, K, N, dt):
    x, w = _x(M, K, dt), _x(N, K, torch.float32, 1) * K ** -0.5
    bias = torch.randn(N, generator=torch.Generator().manual_seed(N))
    pw = ops.pack_w_fp8(w.to(DEV), bias.to(DEV))
    qx, qw = O.dequant(*O.quant_rows(x)), O.dequant(*O.quant(w, 128))
    ref, (A, G), Kb = qx @ qw.t() + bias.double(), _terms(qx, qw), (K + 127) // 128
    A = (A + bias.double().abs(), G)
    y = ops.linear_fp8(x.to(DEV), pw)
    assert y.dtype == dt
    _check(y, ref, A, Kb, dt)
    assert torch.equal(y, ops.linear_fp8(x.to(DEV), pw))                       # the same bits every time
    # operands quantised once, and another output type
    _check(ops.linear_fp8(ops.quantize_fp8(x.to(DEV)), pw, out_dtype=torch.float32), ref, A, Kb, torch.float32)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (5, 129, 64), (64, 320, 200), (130, 96, 333), (300, 256, 128)])
def test_gradients_vs_float64(ops, M, K, N, dt):
    x, gy, w = _x(M, K, dt), _x(M, N, dt, 2), _x(N, K, torch.float32, 1)
    pw = ops.pack_w_fp8(w.to(DEV))
    gx, gw = ops.linear_fp8_bwd(x.to(DEV), gy.to(DEV), pw)
    qw = O.dequant(*O.quant(w, 128))
    g = O.dequant(*O.quant_rows(gy))
    _check(gx, g @ qw, _terms(g, qw.t()), (N + 127) // 128, dt)
    gc, xc = O.dequant(*O.quant_rows(gy.t().contiguous())), O.dequant(*O.quant_rows(x.t().contiguous()))
    assert gw.dtype == torch.float32
    _check(gw, gc @ xc.t(), _terms(gc, xc), (M + 127) // 128, torch.float32)
    only = ops.linear_fp8_bwd(x.to(DEV), gy.to(DEV), pw, want_gw=False)
    assert only[1] is None and torch.equal(only[0], gx)


def test_gradient_against_differences(ops):
    """Inputs on the e4m3 grid with a 448 in every block: quantisation changes nothing, the product is linear and its differences are exact
    gradients up to the counted roundings."""
    g = torch.Generator().manual_seed(0)
    M, K, N = 40, 256, 128

    def grid(r, c):
        t = torch.randint(-8, 9, (r, c), generator=g).float()
        t[:, ::128] = 448.0
        return t
    x, w, gy = grid(M, K), grid(N, K), grid(M, N)
    pw = ops.pack_w_fp8(w.to(DEV))
    gx, _ = ops.linear_fp8_bwd(x.to(DEV), gy.to(DEV), pw, want_gw=False)
    f = lambda t: (ops.linear_fp8(t.to(DEV), pw).double().cpu() * gy.double()).sum(1)      # noqa: E731
    for k in (1, 77, 200):
        xp, xm = x.clone(), x.clone()
        xp[:, k] += 1.0
        xm[:, k] -= 1.0
        ok = (xp[:, k].abs() <= 8) & (xm[:, k].abs() <= 8)          # still on the grid
        # all terms are integers below 2^24 in each output: exact
        assert torch.equal(((f(xp) - f(xm)) / 2)[ok], gx[:, k].double().cpu()[ok])


def test_strides_and_leading_shapes(ops):
    base = _x(6 * 50, 400, torch.float16).reshape(6, 50, 400).to(DEV)
    w = _x(96, 128, torch.float32, 1).to(DEV)
    pw = ops.pack_w_fp8(w)
    want = ops.linear_fp8(base[..., 8:136].contiguous(), pw)
    assert want.shape == (6, 50, 96)
    assert torch.equal(ops.linear_fp8(base[..., 8:136], pw), want)              # a column slice, 16-byte aligned
    odd = base[..., 5:133]
    assert torch.equal(ops.linear_fp8(odd, pw), ops.linear_fp8(odd.contiguous(), pw))        # not aligned
    few = base[0, :20, 5:133]
    assert torch.equal(ops.linear_fp8(few, pw), ops.linear_fp8(few.contiguous(), pw))
    every = base[:, ::2, 8:136].reshape(-1, 128)                                # (reshape copies) against the view of one item
    assert torch.equal(ops.linear_fp8(base[0, ::2, 8:136], pw), ops.linear_fp8(every[:25], pw))
    gy = _x(300, 96, torch.float16, 4).reshape(6, 50, 96).to(DEV)
    for a, b in zip(ops.linear_fp8_bwd(odd, gy, pw), ops.linear_fp8_bwd(odd.contiguous(), gy, pw)):
        assert torch.equal(a, b)
    assert ops.linear_fp8(base[0, 0, 8:136], pw).shape == (96,)


@pytest.mark.parametrize("M", [8, 200])
def test_not_finite_rows_stay_alone(ops, M):
    x = _x(M, 300, torch.float16)
    w = _x(130, 300, torch.float32, 1).to(DEV)
    pw = ops.pack_w_fp8(w)
    want = ops.linear_fp8(x.to(DEV), pw)
    y = x.clone()
    y[2, 140], y[5, 0], y[6, 299] = float("nan"), float("inf"), -float("inf")
    got = ops.linear_fp8(y.to(DEV), pw)
    rows = torch.tensor([i for i in range(M) if i not in (2, 5, 6)])
    assert torch.equal(got.cpu()[rows], want.cpu()[rows])
    assert torch.isnan(got.cpu()[[2, 5, 6]]).all()


def test_extremes_of_range(ops):
    """Blocks whose scale is at the ends of fp32's range: a tiny one keeps its relative precision down to 2^-100, a huge one does not overflow."""
    x = torch.zeros(4, 128)
    x[0], x[1], x[2], x[3, 5] = 2.0 ** -99, 3.0e38, 1e-40, 65504.0
    f = ops.quantize_fp8(x.to(DEV))
    q, s = O.quant_rows(x)
    assert torch.equal(_bytes(f.q), q) and torch.equal(f.scale.cpu().double(), s.t())
    assert torch.isfinite(f.scale).all() and (f.scale > 0).all()


def test_empty_and_no_rows(ops):
    pw = ops.pack_w_fp8(_x(20, 40, torch.float32).to(DEV))
    x = torch.empty(0, 3, 40, dtype=torch.float16, device=DEV)
    assert ops.linear_fp8(x, pw).shape == (0, 3, 20) and ops.quantize_fp8(x).q.shape == (0, 128)
    gx, gw = ops.linear_fp8_bwd(x, torch.empty(0, 3, 20, dtype=torch.float16, device=DEV), pw)
    assert gx.shape == (0, 3, 40) and gw.shape == (20, 40) and (gw == 0).all()


def test_captured_and_replayed_on_a_side_stream(ops):
    pw = ops.pack_w_fp8(_x(256, 320, torch.float32, 1).to(DEV), torch.ones(256, device=DEV))
    xs = [_x(200, 320, torch.float16, i).to(DEV) for i in range(4)]
    gy = _x(200, 256, torch.float16, 9).to(DEV)
    x = xs[0].clone()

    def step(t):
        return (ops.linear_fp8(t, pw), ops.linear_fp8(t[:3], pw)) + ops.linear_fp8_bwd(t, gy, pw)
    want = [step(t) for t in xs]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        side = step(x)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, want[0]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x)
    for i, t in enumerate(xs):
        x.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i
        _ = step(xs[0])                                   # eager work between the replays


def test_a_copied_weight_is_its_own(ops):
    """copy.deepcopy of a model copies the tensors of a packed weight: the copy reads its own bytes, scales and bias."""
    import copy
    x = _x(40, 300, torch.float16).to(DEV)
    pw = ops.pack_w_fp8(_x(200, 300, torch.float32, 1).to(DEV), torch.randn(200).to(DEV))
    y, g = ops.linear_fp8(x, pw), ops.linear_fp8_bwd(x, _x(40, 200, torch.float16, 3).to(DEV), pw)
    other = copy.deepcopy(pw)
    for t in (pw.q, pw.qt, pw.scale, pw.bias):
        t.zero_()
    assert torch.equal(ops.linear_fp8(x, other), y) and not ops.linear_fp8(x, pw).any()
    assert torch.equal(ops.linear_fp8_bwd(x, _x(40, 200, torch.float16, 3).to(DEV), other)[0], g[0])


def test_stored_weights_of_other_layouts(ops):
    """load_w_fp8 takes bytes and scales in any strides."""
    x = _x(40, 300, torch.float16).to(DEV)
    pw = ops.pack_w_fp8(_x(200, 300, torch.float32, 1).to(DEV))
    q = pw.q[:, :300].view(torch.float8_e4m3fn)
    turned = ops.load_w_fp8(q.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn), pw.scale.t().contiguous().t())
    assert torch.equal(turned.q, pw.q) and torch.equal(turned.qt, pw.qt) and torch.equal(turned.scale, pw.scale)
    assert torch.equal(ops.linear_fp8(x, turned), ops.linear_fp8(x, pw))


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("M,K,N", [(600, 2600, 333), (900, 2600, 333), (400, 5120, 640), (257, 3900, 1001)])
def test_slices_of_a_long_reduction(ops, M, K, N, out):
    """Few tiles under a long K axis: its slices' fp32 sums and the bias are added before the one rounding (bound: the sum over the blocks has the same
    additions in another order, and one more per slice, within the 128 of a block counted twice)."""
    h = ops.handle(0)
    sliced = M != 600          # (there one launch of small tiles does it)
    assert (h.lib.tfmq_linear_fp8_ws_bytes(h.h, M, N, K, 1) > 0) == sliced          # (only slices need room for operands that are quantised already)
    x, w, b = _x(M, K, torch.float16), _x(N, K, torch.float32, 1), torch.randn(N, generator=torch.Generator().manual_seed(5))
    pw = ops.pack_w_fp8(w.to(DEV), b.to(DEV))
    y = ops.linear_fp8(x.to(DEV), pw, out)
    assert y.dtype == out and (not sliced or torch.equal(y, ops.linear_fp8(ops.quantize_fp8(x.to(DEV)), pw, out)))
    qx, qw = O.dequant(*O.quant_rows(x)), O.dequant(*O.quant(w, 128))
    A = _terms(qx, qw)
    _check(y, qx @ qw.t() + b.double(), (A[0] + b.double().abs(), A[1]), (K + 127) // 128 + 1, out)


def test_a_packed_bias_is_a_copy(ops):
    """pack_w_fp8 and load_w_fp8 lay a layer out once: an update in place of the bias they were given changes the packed layer no more than one of the weight."""
    x = _x(40, 300, torch.float16).to(DEV)
    w, b = _x(200, 300, torch.float32, 1).to(DEV), torch.randn(200, generator=torch.Generator().manual_seed(3)).to(DEV)
    pw = ops.pack_w_fp8(w, b)
    ld = ops.load_w_fp8(pw.q[:, :300].view(torch.float8_e4m3fn), pw.scale, b)
    y = ops.linear_fp8(x, pw)
    w.zero_()
    b.zero_()
    assert torch.equal(ops.linear_fp8(x, pw), y) and torch.equal(ops.linear_fp8(x, ld), y)
