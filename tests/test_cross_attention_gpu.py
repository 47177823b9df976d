"""K18: ops.cross_attention / cross_attention_bwd against the formulas in 64 bits, per item and head over the kept keys.

Tolerances, u = eps / 2 of the operand type (a rounding is off by at most half a step):
 * forward: p is rounded once (u p, relative), o once (u o); scores, exponentials and sums are fp32.  A score's fp32 error is at most
   (d + 2) 2^-24 sum_c |q_c k_c| scale, which moves p by that relative amount; exp2 and the 1 / l division add 2^-21.  So
       |o - o64| <= (u + e) sum_j p |v| + u |o64| + half the type's smallest step,    e = 2 max_j (d + 2) 2^-24 scale |q| |k| + (Tk + 8) 2^-24 + 2^-21.
   fp16 p below 2^-14 is subnormal: each loses at most 2^-25 absolute, relative to a running maximum's 1: 2^-25 sum_j |v_j| / l, l >= 1.
 * lse: e + 2^-23 |lse|.
 * backward: the forward's o enters D rounded (u sum |o go|), p in dv is rounded (u), ds in dq and dk is rounded (u), results once (u).  With
   a = p (sum_c |go v| + sum_c |o go|) per (i, j):  |dq| error <= scale sum_j (u a + e a + u p sum_c |o go|) |k| + u |dq|, and the same with |q| summed over rows
   for dk; dv error <= sum_i (u + e) p |go| + u |dv|.  fp16 carries ds and p with powers of two, so what underflows is below 2^-25 of the row's
   (slice's) largest |go| times ...: 2^-25 gmax sum |k| (or |q|), and 2^-37 sum |go| in dv.
 * range: an exponential below fp32's smallest normal number 2^-126 is zero (v_exp_f32 has no subnormal results, nor do the operand types keep
   smaller ones), so every p and every ds may be off by 2^-126 absolutely, whatever their relative error.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOW = 2.0 ** -126


@pytest.fixture(scope="module")
def ops():
    import tfmq_dm_amd.ops as ops
    return ops


def _mk(B, Tq, Tk, H, G, d, dt, seed=0, fused=True):
    g = torch.Generator().manual_seed(seed + B + 3 * Tq + 5 * Tk + 7 * H + 11 * G + 13 * d)
    r = lambda *s: torch.randn(*s, generator=g).to(dt)      # noqa: E731
    q, go = r(B, Tq, H * d), r(B, Tq, H * d)
    kv = r(B, Tk, 2 * G * d)
    k, v = (kv[..., :G * d], kv[..., G * d:]) if fused else (kv[..., :G * d].contiguous(), kv[..., G * d:].contiguous())
    return q, k, v, go


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _fused_dev(k, v):
    """k | v on the device as the halves of one buffer, the way a fused projection leaves them."""
    kv = torch.cat([k, v], -1).to(DEV)
    C = k.shape[-1]
    return kv[..., :C], kv[..., C:]


def _ref(q, k, v, H, scale, G=None, q_lens=None, kv_lens=None, mask=None, go=None):
    """64-bit results and their error bounds."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    G = H if G is None else G
    B, Tq, Cq = q.shape
    Tk, d, rep = k.shape[1], Cq // H, H // G
    Z = lambda *s: torch.zeros(*s, dtype=torch.float64)      # noqa: E731
    R = {"o": Z(B, Tq, Cq), "lse": torch.full((B, H, Tq), -math.inf, dtype=torch.float64), "dq": Z(B, Tq, Cq), "dk": Z(B, Tk, G * d), "dv": Z(B, Tk, G * d)}
    E = {n: torch.zeros_like(t) for n, t in R.items()}
    for b in range(B):
        n = Tq if q_lens is None else int(q_lens[b])
        idx = torch.arange(Tk if kv_lens is None else min(max(int(kv_lens[b]), 0), Tk))
        if mask is not None:
            idx = idx[mask[b, idx]]
        if idx.numel() == 0 or n == 0:
            continue
        for h in range(H):
            cq, ck = slice(h * d, (h + 1) * d), slice(h // rep * d, (h // rep + 1) * d)
            qq, kk, vv = q[b, :n, cq].double(), k[b, idx, ck].double(), v[b, idx, ck].double()
            s = qq @ kk.t() * scale
            lse = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[:, None])
            o = p @ vv
            e = (2 * (d + 2) * 2.0 ** -24 * scale * (qq.abs() @ kk.abs().t()).amax(-1) + (idx.numel() + 8) * 2.0 ** -24 + 2.0 ** -21)[:, None]
            R["o"][b, :n, cq], R["lse"][b, h, :n] = o, lse
            E["o"][b, :n, cq] = (u + e) * (p @ vv.abs()) + u * o.abs() + tiny * (1 + vv.abs().sum(0)) + LOW * vv.abs().sum(0)
            E["lse"][b, h, :n] = e[:, 0] + 2.0 ** -23 * lse.abs()
            if go is None:
                continue
            gg = go[b, :n, cq].double()
            dp, D, Da = gg @ vv.t(), (o * gg).sum(-1, keepdim=True), (o.abs() * gg.abs()).sum(-1, keepdim=True)
            ds = p * (dp - D)
            Ea = ((u + e) * p + LOW) * (gg.abs() @ vv.abs().t() + Da) + u * p * Da + LOW
            gm = gg.abs().amax()
            und = tiny * gg.abs().amax(-1, keepdim=True)
            R["dq"][b, :n, cq] = scale * ds @ kk
            E["dq"][b, :n, cq] = scale * ((Ea + und) @ kk.abs()) + u * R["dq"][b, :n, cq].abs() + tiny
            dk, dv = scale * ds.t() @ qq, p.t() @ gg
            R["dk"][b, idx, ck] += dk
            R["dv"][b, idx, ck] += dv
            E["dk"][b, idx, ck] += scale * ((Ea + tiny * gm).t() @ qq.abs())
            E["dv"][b, idx, ck] += ((u + e) * p + LOW).t() @ gg.abs() + tiny * 2.0 ** -12 * gg.abs().sum(0)
    for n in ("dk", "dv"):
        E[n] += u * R[n].abs() + tiny
    return R, E


def _check(name, got, R, E):
    got, ref, err = got.double().cpu(), R[name], E[name]
    assert got.shape == ref.shape, name
    if name == "lse":
        empty = torch.isinf(ref)
        assert torch.equal(torch.isinf(got) & (got < 0), empty)
        got, ref, err = got[~empty], ref[~empty], err[~empty]
    assert torch.isfinite(got).all(), name
    bad = (got - ref).abs() > err
    assert not bad.any(), (name, int(bad.sum()), float(((got - ref).abs() / err.clamp_min(1e-300)).max()))


def _run(ops, q, k, v, go, H, scale, G=None, q_lens=None, kv_lens=None, mask=None, check=True):
    how = dict(kv_heads=G, **dict(zip(("q_lens", "kv_lens", "mask"), _dev(q_lens, kv_lens, mask))))
    qd, gd = _dev(q, go)
    kd, vd = _fused_dev(k, v)
    o, lse = ops.cross_attention(qd, kd, vd, H, scale, want_lse=True, **how)
    assert torch.equal(o, ops.cross_attention(qd, kd, vd, H, scale, **how))
    grads = ops.cross_attention_bwd(qd, kd, vd, o, lse, gd, H, scale, **how)
    again = ops.cross_attention_bwd(qd, kd, vd, o, lse, gd, H, scale, **how)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))          # the same bits every time
    if check:
        R, E = _ref(q, k, v, H, scale, G, q_lens, kv_lens, mask, go)
        for n, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse) + tuple(grads)):
            assert t.dtype == (torch.float32 if n == "lse" else q.dtype)
            _check(n, t, R, E)
    return (o, lse) + tuple(grads)


TYPES = [torch.float16, torch.bfloat16]


# every bucket of head dims and sizes inside one; lengths of one, tile edges (64 keys, 128 rows) and odd ones
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,Tq,Tk,H,d", [(1, 1, 1, 1, 8), (2, 5, 7, 2, 32), (2, 128, 77, 8, 40), (1, 129, 64, 3, 64), (2, 33, 65, 2, 72), (1, 200, 128, 4, 80),
                                         (1, 70, 129, 2, 96), (2, 31, 200, 2, 120), (1, 65, 300, 2, 128), (1, 40, 100, 2, 136), (2, 130, 77, 2, 160)])
def test_plain(ops, B, Tq, Tk, H, d, dt):
    q, k, v, go = _mk(B, Tq, Tk, H, H, d, dt)
    _run(ops, q, k, v, go, H, d ** -0.5)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,G,Tq", [(8, 1, 1), (8, 2, 3), (6, 3, 50), (4, 2, 129), (32, 8, 1)])
def test_shared_key_heads(ops, H, G, Tq, dt):
    q, k, v, go = _mk(2, Tq, 150, H, G, 64, dt)
    _run(ops, q, k, v, go, H, 0.125, G)


@pytest.mark.parametrize("dt", TYPES)
def test_lengths_and_masks(ops, dt):
    B, Tq, Tk, H, G, d = 6, 37, 150, 4, 2, 40
    q, k, v, go = _mk(B, Tq, Tk, H, G, d, dt)
    g = torch.Generator().manual_seed(5)
    mask = torch.rand(B, Tk, generator=g) < 0.5
    mask[1] = False                                   # an item that keeps nothing
    mask[2, :64] = False                              # its first tile keeps nothing
    mask[3] = False
    mask[3, 100] = True                               # one key
    kv_lens = torch.tensor([150, 150, 149, 128, 0, 1], dtype=torch.int32)
    mask[5, 0] = True
    q_lens = torch.tensor([37, 36, 1, 37, 20, 0], dtype=torch.int32)
    for ql in (None, q_lens):
        for kl in (None, kv_lens):
            for m in (None, mask):
                _run(ops, q, k, v, go, H, d ** -0.5, G, ql, kl, m)
    # a length outside [0, Tk] is clamped
    wild = torch.tensor([1000, -5, 149, 128, 0, 1], dtype=torch.int32)
    tame = torch.tensor([150, 0, 149, 128, 0, 1], dtype=torch.int32)
    for a, b in zip(_run(ops, q, k, v, go, H, 0.2, G, None, wild, mask, check=False), _run(ops, q, k, v, go, H, 0.2, G, None, tame, mask)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 65504.0])
def test_what_dropped_places_hold_is_not_seen(ops, bad):
    B, Tq, Tk, H, d = 3, 40, 100, 2, 64
    q, k, v, go = _mk(B, Tq, Tk, H, H, d, torch.float16)
    kv_lens = torch.tensor([100, 70, 0], dtype=torch.int32)
    q_lens = torch.tensor([40, 30, 40], dtype=torch.int32)
    mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(1)) < 0.7
    want = _run(ops, q, k, v, go, H, 0.125, None, q_lens, kv_lens, mask)
    k, v, q, go = k.clone(), v.clone(), q.clone(), go.clone()
    for b in range(B):
        drop = ~mask[b]
        drop[int(kv_lens[b]):] = True
        k[b, drop], v[b, drop] = bad, bad
        q[b, int(q_lens[b]):], go[b, int(q_lens[b]):] = bad, bad
    for a, b in zip(want, _run(ops, q, k, v, go, H, 0.125, None, q_lens, kv_lens, mask, check=False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", TYPES)
def test_peaked_and_far_scores(ops, dt):
    """Rows whose softmax is one key, scores far from zero on both sides, and a running maximum that rises tile after tile."""
    B, Tq, Tk, H, d = 1, 48, 400, 2, 64
    q, k, v, go = _mk(B, Tq, Tk, H, H, d, dt)
    k = (k.float() * (1 + torch.arange(Tk).float()[None, :, None] / 40)).to(dt)
    q = (q.float() * 4).to(dt)
    _run(ops, q, k, v, go, H, 0.5)


def test_small_gradients_keep_their_precision_in_fp16(ops):
    """go of 2^-12 averaged over 4000 states: ds lies below fp16's normal numbers."""
    q, k, v, go = _mk(1, 64, 4000, 2, 2, 64, torch.float16)
    go = (go.float() * 2.0 ** -12).to(torch.float16)
    o, lse, dq, dk, dv = _run(ops, q, k, v, go, 2, 0.125)
    R, _ = _ref(q, k, v, 2, 0.125, go=go)
    # rounding to fp16 of results that are themselves subnormal is the only loss: at most half of 2^-24 each
    for n, t in (("dq", dq), ("dv", dv)):
        err = (t.double().cpu() - R[n]).abs().max()
        assert err <= 2.0 ** -25 + 4 * 2.0 ** -11 * R[n].abs().max(), n


def test_slices_of_a_long_axis(ops):
    """Few rows over many states (the key axis is cut), and few states under many rows (the row axis is cut in the gradients)."""
    h = ops.handle(0)
    assert h.lib.tfmq_xattn_splits(h.h, 2, 8, 2, 1, 5000) > 1 and h.lib.tfmq_xattn_bwd_splits(h.h, 1, 4, 4, 3000, 77) > 1
    q, k, v, go = _mk(2, 1, 5000, 8, 2, 64, torch.bfloat16)
    _run(ops, q, k, v, go, 8, 0.125, 2, None, torch.tensor([5000, 100], dtype=torch.int32))
    q, k, v, go = _mk(3, 2, 1030, 4, 4, 128, torch.float16)
    mask = torch.zeros(3, 1030, dtype=torch.bool)
    mask[0], mask[1, 900:905] = True, True
    _run(ops, q, k, v, go, 4, 0.1, None, torch.tensor([2, 1, 2], dtype=torch.int32), None, mask)
    q, k, v, go = _mk(1, 3000, 77, 4, 4, 40, torch.float16)
    _run(ops, q, k, v, go, 4, 0.2, None, torch.tensor([2999], dtype=torch.int32))


def test_gradient_against_differences(ops):
    """Central differences of the 64-bit forward at the kernel's inputs agree with the kernel's gradients within its own bounds plus the
    difference's truncation, h^2 / 6 of a third derivative that is at most 6 (scale |k|)^3 |go| |v| summed."""
    q, k, v, go = _mk(1, 6, 9, 2, 1, 16, torch.bfloat16)
    scale = 0.25
    _, _, dq, dk, dv = _run(ops, q, k, v, go, 2, scale, 1)
    _, E = _ref(q, k, v, 2, scale, 1, go=go)
    h = 2.0 ** -12

    def f(q, k, v):
        R, _ = _ref64(q, k, v, 2, scale, 1)
        return (R * go.double()).sum()

    def _ref64(q, k, v, H, scale, G):
        d = q.shape[-1] // H
        o = torch.zeros_like(q)
        for hd in range(H):
            p = torch.softmax(q[0, :, hd * d:(hd + 1) * d] @ k[0].t() * scale, -1)
            o[0, :, hd * d:(hd + 1) * d] = p @ v[0]
        return o, None
    base = [t.double() for t in (q, k, v)]
    for which, (got, name) in enumerate(((dq, "dq"), (dk, "dk"), (dv, "dv"))):
        for pos in ((0, 0, 0), (0, 3, 5), (0, 5, 15)):
            xs = [t.clone() for t in base]
            xs[which][pos] += h
            up = f(*xs)
            xs[which][pos] -= 2 * h
            fd = (up - f(*xs)) / (2 * h)
            kmax = max(float(t.abs().max()) for t in base) * scale
            trunc = h * h * (kmax ** 3) * float(go.abs().double().sum()) * float(base[2].abs().max())
            assert abs(float(got[pos]) - float(fd)) <= float(E[name][pos]) + trunc, (name, pos)


def test_strides_and_broadcasts(ops):
    B, Tq, Tk, H, d = 3, 20, 70, 2, 40
    q, k, v, go = _dev(*_mk(B, Tq, Tk, H, H, d, torch.float16, fused=False))
    C = H * d
    want, lse = ops.cross_attention(q, k, v, H, 0.2, want_lse=True)
    # a padded row stride, a transposed batch / token order, every second token
    wide = torch.zeros(B, Tq, C + 24, dtype=q.dtype, device=DEV)
    wide[..., 8:8 + C] = q
    assert torch.equal(ops.cross_attention(wide[..., 8:8 + C], k, v, H, 0.2), want)
    tb = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.cross_attention(tb, k, v, H, 0.2), want)
    k2 = torch.zeros(B, 2 * Tk, C, dtype=q.dtype, device=DEV)
    k2[:, ::2] = k
    assert torch.equal(ops.cross_attention(q, k2[:, ::2], v, H, 0.2), want)
    go2 = torch.zeros_like(wide)
    go2[..., 16:16 + C] = go
    for a, b in zip(ops.cross_attention_bwd(wide[..., 8:8 + C], k2[:, ::2], v, want, lse, go2[..., 16:16 + C], H, 0.2),
                    ops.cross_attention_bwd(q, k, v, want, lse, go, H, 0.2)):
        assert torch.equal(a, b)
    # one encoder state set and one mask for the whole batch
    ke, ve, me = k[:1].expand(B, -1, -1), v[:1].expand(B, -1, -1), (torch.arange(Tk, device=DEV) % 3 != 0)[None].expand(B, -1)
    full = ops.cross_attention(q, ke.contiguous(), ve.contiguous(), H, 0.2, mask=me.contiguous())
    assert torch.equal(ops.cross_attention(q, ke, ve, H, 0.2, mask=me), full)


def test_no_states_and_no_queries(ops):
    q, k = torch.ones(2, 3, 64, dtype=torch.float16, device=DEV), torch.ones(2, 0, 64, dtype=torch.float16, device=DEV)
    o, lse = ops.cross_attention(q, k, k, 2, 1.0, want_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = ops.cross_attention_bwd(q, k, k, o, lse, q, 2, 1.0)
    assert (dq == 0).all() and dk.shape == (2, 0, 64) and dv.shape == (2, 0, 64)
    none = torch.ones(2, 0, 64, dtype=torch.float16, device=DEV)
    assert ops.cross_attention(none, q, q, 2, 1.0).shape == (2, 0, 64)
    dq, dk, dv = ops.cross_attention_bwd(none, q, q, none, torch.ones(2, 2, 0, device=DEV), none, 2, 1.0)
    assert (dk == 0).all() and (dv == 0).all()


def test_offsets_beyond_32_bits(ops):
    """A state buffer whose last item begins past 2^31 elements (an item stride, not a dense tensor: 4.4 GB of bf16 are allocated, little is read)."""
    B, Tk, C = 3, 80, 64
    buf = torch.empty((1 << 31) + Tk * 2 * C + 64, dtype=torch.bfloat16, device=DEV)
    stride = 1 << 30
    kv = torch.as_strided(buf, (B, Tk, 2 * C), (stride, 2 * C, 1))
    g = torch.Generator().manual_seed(3)
    small = torch.randn(B, Tk, 2 * C, generator=g).bfloat16().to(DEV)
    kv.copy_(small)
    q = torch.randn(B, 5, C, generator=g).bfloat16().to(DEV)
    want, lse = ops.cross_attention(q, small[..., :C], small[..., C:], 2, 0.2, want_lse=True)
    assert torch.equal(ops.cross_attention(q, kv[..., :C], kv[..., C:], 2, 0.2), want)
    for a, b in zip(ops.cross_attention_bwd(q, kv[..., :C], kv[..., C:], want, lse, q, 2, 0.2),
                    ops.cross_attention_bwd(q, small[..., :C], small[..., C:], want, lse, q, 2, 0.2)):
        assert torch.equal(a, b)


def test_two_captured_graphs_and_eager_work(ops):
    B, Tq, Tk, H, G, d = 2, 1, 2000, 8, 2, 64
    sets = [_dev(*_mk(B, Tq, Tk, H, G, d, torch.bfloat16, seed=i, fused=False)) for i in range(3)]
    wide = [_dev(*_mk(1, 2500, 77, 4, 4, 40, torch.float16, seed=i, fused=False)) for i in range(3)]
    lens = torch.tensor([2000, 700], dtype=torch.int32, device=DEV)

    def one(q, k, v, go):
        o, lse = ops.cross_attention(q, k, v, H, 0.125, G, kv_lens=lens, want_lse=True)
        return (o, lse) + tuple(ops.cross_attention_bwd(q, k, v, o, lse, go, H, 0.125, G, kv_lens=lens))

    def two(q, k, v, go):
        o, lse = ops.cross_attention(q, k, v, 4, 0.2, want_lse=True)
        return (o, lse) + tuple(ops.cross_attention_bwd(q, k, v, o, lse, go, 4, 0.2))
    want1, want2 = [one(*s) for s in sets], [two(*s) for s in wide]
    in1, in2 = [t.clone() for t in sets[0]], [t.clone() for t in wide[0]]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        side = one(*in1)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, want1[0]))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = one(*in1)
    with torch.cuda.graph(g2):
        out2 = two(*in2)
    for i in (0, 1, 2, 0):
        for a, b in zip(in1, sets[i]):
            a.copy_(b)
        for a, b in zip(in2, wide[i]):
            a.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            g2.replay()
        g1.replay()
        _ = one(*sets[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out1, want1[i])), i
        assert all(torch.equal(a, b) for a, b in zip(out2, want2[i])), i


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Tq,Tk,H,G,d", [(1709, 18, 4, 4, 160), (64, 7, 8, 2, 40), (300, 33, 4, 4, 64), (5, 2, 16, 4, 80)])
def test_few_states_lose_only_the_roundings(ops, Tq, Tk, H, G, d, dt):
    """Few kept states leave ds = p (dp - D) small against D.  dq and dk round twice, the ds operand and the result: a rounding's error is at most uniform
    over half a step of eps |x|, rms eps / (2 sqrt 3) of the value, two independent ones sqrt 2 of that (the sum over channels or rows does not add: its
    terms' errors are as independent as its terms)."""
    q, k, v, go = _mk(2, Tq, Tk, H, G, d, dt, Tk)
    lens = torch.tensor([Tk, max(1, Tk // 2)], dtype=torch.int32)
    mask = torch.rand(2, Tk, generator=torch.Generator().manual_seed(Tk)) < 0.6
    mask[:, 0] = True
    o, lse, dq, dk, dv = _run(ops, q, k, v, go, H, d ** -0.5, G, None, lens, mask)
    R, _ = _ref(q, k, v, H, d ** -0.5, G, None, lens, mask, go=go)
    for n, t in (("dq", dq), ("dk", dk)):
        assert float((t.double().cpu() - R[n]).norm() / R[n].norm()) <= 2 ** 0.5 * torch.finfo(dt).eps / (2 * 3 ** 0.5), n
