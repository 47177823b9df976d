"""K17's large products, each case with the kernel that it reaches asserted: the 128 x 128 tiles (few, many, more than the card holds at once), the
256 x 256 tiles, and both gradients in one launch.  Oracle and bounds are those of test_linear_fp8_gpu, at all columns of some rows and all rows of some
columns."""
import pytest
import torch

import _fp8_oracle as O
from test_linear_fp8_gpu import DEV, TYPES, _check, _terms, _x

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import tfmq_dm_amd.ops as ops
    return ops


def _cdiv(a, b):
    return (a + b - 1) // b


def _route(M, K, N, dt, cu):
    """The kernel that multiplies M x K by K x N, by the rules stated in fp8_block.hip."""
    if M <= 32 or _cdiv(M, 32) * _cdiv(N, 32) <= (1 if K > 19 * 128 else 2) * cu:
        return "small"
    nt, kb = _cdiv(M, 128) * _cdiv(N, 128), _cdiv(K, 128)
    if min(cu // nt, kb // 10) > 1:
        return "slices"
    n2 = _cdiv(M, 256) * _cdiv(N, 256)
    if dt != F32 and n2 >= cu and n2 * 4 >= _cdiv(n2, cu) * cu * 3:
        return "256 walk" if n2 > cu else "256"
    return "128 deep" if nt <= cu else "128 walk" if nt > 2 * cu else "128"


def _rows(n):
    """Rows beside the borders of 32, 128 and 256, the last ones, and some between."""
    edge = [i for b in (0, 32, 128, 256, 512, n // 256 * 256, n // 128 * 128, n) for i in (b - 1, b, b + 1)]
    some = torch.randint(0, n, (24,), generator=torch.Generator().manual_seed(n)).tolist()
    return torch.tensor(sorted({i for i in edge + some if 0 <= i < n}))


def _check_product(y, a, b, bias, Kb, dt, what):
    """y against a b^T + bias, a and b the values of the quantised operands."""
    for ra, rb in ((_rows(a.shape[0]), slice(None)), (slice(None), _rows(b.shape[0]))):
        qa, qb = a[ra], b[rb]
        ref, (A, G) = qa @ qb.t(), _terms(qa, qb)
        if bias is not None:
            ref, A = ref + bias[rb].double(), A + bias[rb].double().abs()
        _check(y[ra][:, rb], ref, (A, G), Kb, dt)


CASES = [
    (1024, 520, 640, F16, True, "128 deep"), (1100, 520, 641, BF16, False, "128 deep"), (1100, 200, 1000, F32, True, "128 deep"),
    (4100, 200, 1100, BF16, True, "128"), (4096, 384, 1152, F16, False, "128"), (4100, 640, 1101, F32, False, "128"),
    (8200, 100, 1300, F16, True, "128 walk"), (8200, 384, 1301, BF16, False, "128 walk"), (8192, 1280, 1408, F16, False, "128 walk"),
    (8192, 320, 2560, BF16, True, "128 walk"), (8200, 384, 1300, F32, True, "128 walk"),
    (4096, 384, 4096, F16, False, "256"), (4000, 1290, 4090, BF16, True, "256"),
    (5000, 128, 5100, F16, True, "256 walk"), (5000, 260, 5101, BF16, True, "256 walk"), (5120, 384, 5120, F16, False, "256 walk"), (5000, 1280, 5100, F16, False, "256 walk"),
]


@pytest.mark.parametrize("M,K,N,dt,with_bias,route", CASES)
def test_large_products(ops, M, K, N, dt, with_bias, route):
    assert _route(M, K, N, dt, torch.cuda.get_device_properties(0).multi_processor_count) == route
    x, w = _x(M, K, dt), _x(N, K, F32, 1) * K ** -0.5
    bias = torch.randn(N, generator=torch.Generator().manual_seed(N)) if with_bias else None
    pw = ops.pack_w_fp8(w.to(DEV), None if bias is None else bias.to(DEV))
    y = ops.linear_fp8(x.to(DEV), pw)
    assert y.dtype == dt
    _check_product(y.cpu(), O.dequant(*O.quant_rows(x)), O.dequant(*O.quant(w, 128)), bias, _cdiv(K, 128), dt, route)
    assert torch.equal(y, ops.linear_fp8(x.to(DEV), pw))                                      # the same bits every time,
    assert torch.equal(y, ops.linear_fp8(ops.quantize_fp8(x.to(DEV)), pw))                    # and from operands that are quantised already


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N,route", [(1333, 1000, 777, "128 deep"), (2100, 640, 520, "128 deep"), (5000, 1030, 129, "128"), (9000, 1024, 257, "128 walk"),
                                         (4000, 4090, 200, "256")])
def test_large_gradients(ops, M, K, N, route, dt):
    got = _route(M, N, K, dt, torch.cuda.get_device_properties(0).multi_processor_count)          # (of x's gradient: reduced over N)
    assert got == (route if dt != F32 or route != "256" else "128 walk")
    x, gy, w = _x(M, K, dt), _x(M, N, dt, 2), _x(N, K, F32, 1)
    pw = ops.pack_w_fp8(w.to(DEV))
    xd, gd = x.to(DEV), gy.to(DEV)
    gx, gw = ops.linear_fp8_bwd(xd, gd, pw)
    _check_product(gx.cpu(), O.dequant(*O.quant_rows(gy)), O.dequant(*O.quant(w, 128)).t().contiguous(), None, _cdiv(N, 128), dt, route)
    gc, xc = O.dequant(*O.quant_rows(gy.t().contiguous())), O.dequant(*O.quant_rows(x.t().contiguous()))
    _check_product(gw.cpu(), gc, xc, None, _cdiv(M, 128), F32, "gw")
    again = ops.linear_fp8_bwd(xd, gd, pw)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)
    assert torch.equal(ops.linear_fp8_bwd(xd, gd, pw, want_gw=False)[0], gx)
    assert torch.equal(ops.linear_fp8_bwd(xd, gd, pw, want_gx=False)[1], gw)


def test_large_products_replayed(ops):
    """Both tile forms and the gradients' launch in one captured graph, other inputs at each replay, eager work between."""
    pw, pb = ops.pack_w_fp8(_x(1300, 200, F32, 1).to(DEV), torch.ones(1300, device=DEV)), ops.pack_w_fp8(_x(4090, 130, F32, 2).to(DEV))
    xs = [_x(8200, 200, F16, i).to(DEV) for i in range(3)]
    bs = [_x(4000, 130, BF16, i).to(DEV) for i in range(3)]
    gy = _x(8200, 1300, F16, 9).to(DEV)
    x, b = xs[0].clone(), bs[0].clone()

    def step(t, u):
        return (ops.linear_fp8(t, pw), ops.linear_fp8(u, pb)) + ops.linear_fp8_bwd(t, gy, pw)
    want = [step(t, u) for t, u in zip(xs, bs)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(x, b)
    for i in (0, 1, 2, 1):
        x.copy_(xs[i])
        b.copy_(bs[i])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i])), i
        _ = step(xs[0], bs[0])
        torch.cuda.synchronize()


@pytest.mark.parametrize("dx,dg", [(F32, F16), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("M,K,N", [(40, 200, 96), (1333, 1000, 777)])
def test_gradients_of_mixed_types(ops, M, K, N, dx, dg):
    """x and gy of different types: gx in gy's, gw in fp32."""
    x, gy, w = _x(M, K, dx), _x(M, N, dg, 2), _x(N, K, F32, 1)
    pw = ops.pack_w_fp8(w.to(DEV))
    gx, gw = ops.linear_fp8_bwd(x.to(DEV), gy.to(DEV), pw)
    assert gx.dtype == dg and gw.dtype == F32
    _check_product(gx.cpu(), O.dequant(*O.quant_rows(gy)), O.dequant(*O.quant(w, 128)).t().contiguous(), None, _cdiv(N, 128), dg, "gx")
    _check_product(gw.cpu(), O.dequant(*O.quant_rows(gy.t().contiguous())), O.dequant(*O.quant_rows(x.t().contiguous())), None, _cdiv(M, 128), F32, "gw")


@pytest.mark.parametrize("out", [F16, F32])
def test_other_output_types_of_large_products(ops, out):
    for M, K, N in ((1100, 300, 1000), (4100, 300, 1100), (4000, 130, 4090)):
        x, w = _x(M, K, BF16), _x(N, K, F32, 1)
        y = ops.linear_fp8(x.to(DEV), ops.pack_w_fp8(w.to(DEV)), out)
        assert y.dtype == out
        _check_product(y.cpu(), O.dequant(*O.quant_rows(x)), O.dequant(*O.quant(w, 128)), None, _cdiv(K, 128), out, (M, K, N))


def test_more_than_2_to_the_31_elements(ops):
    """Rows on both sides of 2^31 elements of x, y, gy and gx, and the weight's gradient over all of them."""
    M, K, N = (1 << 31) // 640 + 1000, 640, 648
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty(M, K, dtype=BF16, device=DEV)
    x[:] = torch.randn(1024, K, device=DEV, generator=g).to(BF16).repeat(_cdiv(M, 1024), 1)[:M]
    w = torch.randn(N, K, device=DEV, generator=g)
    pw = ops.pack_w_fp8(w)
    at = torch.tensor([0, 1000, (1 << 31) // 648, (1 << 31) // 640, (1 << 31) // 640 + 1, M - 1000, M - 1])
    rows = x[at.to(DEV)].cpu()
    y = ops.linear_fp8(x, pw)
    qw = O.dequant(*O.quant(w.cpu(), 128))
    qx = O.dequant(*O.quant_rows(rows))
    _check(y[at.to(DEV)], qx @ qw.t(), _terms(qx, qw), 5, BF16)
    gx, gw = ops.linear_fp8_bwd(x, y, pw)
    gy = y[at.to(DEV)].cpu()
    qg = O.dequant(*O.quant_rows(gy))
    _check(gx[at.to(DEV)], qg @ qw, _terms(qg, qw.t()), 6, BF16)
    # every block of 128 tokens is one of eight (the rows repeat after 1024), the last one ragged
    ref, A = torch.zeros(N, K, dtype=torch.float64), torch.zeros(N, K, dtype=torch.float64)
    full, rest = M // 128, M % 128
    for i in range(8):
        for r0, n, times in ((i * 128, 128, (full - i + 7) // 8), (full % 8 * 128, rest, 1 if i == 0 and rest else 0)):
            if times:
                gc = O.dequant(*O.quant_rows(y[r0:r0 + n].cpu().t().contiguous()))
                xc = O.dequant(*O.quant_rows(x[r0:r0 + n].cpu().t().contiguous()))
                ref, A = ref + times * (gc @ xc.t()), A + times * (gc.abs() @ xc.abs().t())
    _check(gw, ref, (A, A * 0), _cdiv(M, 128), F32)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", [(20000, 1, 1), (20000, 130, 7), (17000, 64, 33), (40, 1 << 20, 40), (2, 1 << 22, 3)])
def test_ends_of_the_sizes(ops, M, K, N, dt):
    """One column or channel under many rows, and the longest reductions."""
    x, w = _x(M, K, dt), _x(N, K, F32, 1) * K ** -0.5
    pw = ops.pack_w_fp8(w.to(DEV))
    y = ops.linear_fp8(x.to(DEV), pw)
    _check_product(y.cpu(), O.dequant(*O.quant_rows(x)), O.dequant(*O.quant(w, 128)), None, _cdiv(K, 128), dt, (M, K, N))
    if M * K > 1 << 22:
        return
    gy = _x(M, N, dt, 2)
    gx, gw = ops.linear_fp8_bwd(x.to(DEV), gy.to(DEV), pw)
    _check_product(gx.cpu(), O.dequant(*O.quant_rows(gy)), O.dequant(*O.quant(w, 128)).t().contiguous(), None, _cdiv(N, 128), dt, "gx")
    _check_product(gw.cpu(), O.dequant(*O.quant_rows(gy.t().contiguous())), O.dequant(*O.quant_rows(x.t().contiguous())), None, _cdiv(M, 128), F32, "gw")
