"""K18 where it can go wrong: values that are not finite, the range of the fp16 gradients, few kept states in a long buffer, long tails.

Bounds, u = eps / 2 of the operand type, n kept states, f = e + (d + n + 8) 2^-24 with e the score's share (test_cross_attention_gpu):
 * o: (u + e) sum p |v| + u |o|; fp16 probabilities are carried with 2^7, so one below 2^-21 of the row's largest loses at most 2^-32 of it.
 * D = sum_j p_j dp_j in fp32: with a_j = sum_c |go v_j|, A = sum_j p_j a_j its error is at most 2 f A, that of ds = p (dp - D) before its rounding
   3 f p (a + A).  ds is rounded once to the operand type (u |ds|).  Over more than 128 states the walk starts from the D0 of the rounded o,
   |D - D0| <= (u + 2 f) A, and the difference is put right with p rounded: 2 u (u + 2 f) A p more.
 * fp16 carries ds with a power of two by the row's (dq) or slice's (dk) largest |dp - D|: what underflows is below 2^-33 of that.
 * results are rounded once more; sums over n states or m rows in fp32 add n (m) 2^-24 of their terms' magnitudes.
"""
import math

import pytest
import torch

from test_cross_attention_gpu import DEV, TYPES, _check, _dev, _fused_dev, _mk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import tfmq_dm_amd.ops as ops
    return ops


def _exact(q, k, v, go, H, scale, G=None, kv_lens=None, mask=None, late=None):
    """64-bit results and the bounds above (late: whether D is put right afterwards)."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    half = dt == torch.float16
    tiny = 2.0 ** -25 if half else 0.0
    G = H if G is None else G
    (B, Tq, Cq), Tk, rep = q.shape, k.shape[1], H // G
    d = Cq // H
    Z = lambda *s: torch.zeros(*s, dtype=torch.float64)      # noqa: E731
    R = {"o": Z(B, Tq, Cq), "lse": torch.full((B, H, Tq), -math.inf, dtype=torch.float64), "dq": Z(B, Tq, Cq), "dk": Z(B, Tk, G * d), "dv": Z(B, Tk, G * d)}
    E = {n: torch.zeros_like(t) for n, t in R.items()}
    for b in range(B):
        idx = torch.arange(Tk if kv_lens is None else int(kv_lens[b]))
        if mask is not None:
            idx = idx[mask[b, idx]]
        n = idx.numel()
        if n == 0:
            continue
        for h in range(H):
            cq, ck = slice(h * d, (h + 1) * d), slice(h // rep * d, (h // rep + 1) * d)
            qq, kk, vv, gg = q[b, :, cq].double(), k[b, idx, ck].double(), v[b, idx, ck].double(), go[b, :, cq].double()
            s = qq @ kk.t() * scale
            lse = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[:, None])
            o = p @ vv
            e = (2 * (d + 2) * 2.0 ** -24 * scale * (qq.abs() @ kk.abs().t()).amax(-1) + (n + 8) * 2.0 ** -24 + 2.0 ** -21)[:, None]
            f = e + (d + n + 8) * 2.0 ** -24
            R["o"][b, :, cq], R["lse"][b, h] = o, lse
            E["o"][b, :, cq] = (u + e) * (p @ vv.abs()) + u * o.abs() + tiny + (2.0 ** -32 if half else 2.0 ** -126) * vv.abs().sum(0)
            E["lse"][b, h] = e[:, 0] + 2.0 ** -23 * lse.abs()
            dp, a = gg @ vv.t(), gg.abs() @ vv.abs().t()
            A, diff = (p * a).sum(-1, keepdim=True), dp - (p * dp).sum(-1, keepdim=True)
            ds, low = p * diff, 2.0 ** -126 * (a + (p * a).sum(-1, keepdim=True))
            und = 2.0 ** -33 * diff.abs() if half else torch.zeros_like(diff)
            Ed = u * ds.abs() + 3 * f * p * (a + A) + low
            more = 2 * u * (u + 2 * f) * A * p + (u * A * 2.0 ** -25 if half else 0.0) if (Tk > 128 if late is None else late) else 0.0
            R["dq"][b, :, cq] = scale * ds @ kk
            E["dq"][b, :, cq] = scale * (Ed + more + und.amax(-1, keepdim=True) + n * 2.0 ** -24 * ds.abs()) @ kk.abs() + tiny
            R["dk"][b, idx, ck] += scale * ds.t() @ qq
            R["dv"][b, idx, ck] += p.t() @ gg
            E["dk"][b, idx, ck] += scale * (Ed + und.amax() + rep * Tq * 2.0 ** -24 * ds.abs()).t() @ qq.abs()
            E["dv"][b, idx, ck] += ((u + e + rep * Tq * 2.0 ** -24) * p + 2.0 ** -126).t() @ gg.abs() + tiny * 2.0 ** -12 * gg.abs().sum(0)
    E["dq"] += u * R["dq"].abs()
    for n in ("dk", "dv"):
        E[n] += u * R[n].abs() + tiny
    return R, E


def _all(ops, q, k, v, go, H, scale, G=None, kv_lens=None, mask=None):
    """(o, lse, dq, dk, dv) on the device; the same bits (NaN counted as equal) from a second call."""
    how = dict(kv_heads=G, **dict(zip(("kv_lens", "mask"), _dev(kv_lens, mask))))
    (qd, gd), (kd, vd) = _dev(q, go), _fused_dev(k, v)

    def once():
        o, lse = ops.cross_attention(qd, kd, vd, H, scale, want_lse=True, **how)
        return dict(zip(("o", "lse", "dq", "dk", "dv"), (o, lse) + tuple(ops.cross_attention_bwd(qd, kd, vd, o, lse, gd, H, scale, **how))))
    got, again = once(), once()
    for n in got:
        _same(got[n], again[n], n)
    return got


def _same(a, b, what):
    a, b = a.float().cpu(), b.float().cpu()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)), what


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("dt", TYPES)
def test_c_entry_without_states(ops, dt, splits):
    """tfmq_xattn_fwd takes Tk = 0 with k and v null: zeros and -inf, nothing read."""
    B, H, Tq, d = 2, 3, 5, 40
    q = torch.ones(B, Tq, H * d, dtype=dt, device=DEV)
    o, lse = torch.full_like(q, 7.0), torch.zeros(B, H, Tq, device=DEV)
    ws = torch.empty(splits * B * H * Tq * (d + 2), device=DEV)
    h = ops.handle(0)
    desc = ops._XATTN.pack(ops._DT_CODE[dt], B, H, H, Tq, 0, d, 1.0, q.data_ptr(), 0, 0, Tq * H * d, H * d, 0, 0, 0, 0, 0, 0, 0, 0, o.data_ptr(), 0, 0,
                           lse.data_ptr(), 0, 0, 0, 0, 0, 0, ws.data_ptr(), splits)
    h.call("xattn_fwd", desc, ops._stream(0))
    assert (o == 0).all() and (lse == -math.inf).all()


BAD = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("where", ["q", "go"])
@pytest.mark.parametrize("Tq,Tk", [(40, 100), (40, 200), (3000, 100)])
def test_dropped_keys_have_zero_gradients_whatever_live_rows_hold(ops, Tq, Tk, where, bad):
    """A live row that is not finite (a loss scale too large) spoils the kept keys of its item; masked ones and those behind the length stay zero, with
    the rows in one slice or in several."""
    B, H, d = 3, 2, 64
    h = ops.handle(0)
    assert Tq < 3000 or h.lib.tfmq_xattn_bwd_splits(h.h, B, H, H, Tq, Tk) > 1
    q, k, v, go = _mk(B, Tq, Tk, H, H, d, torch.float16)
    mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(1)) < 0.7
    kv_lens = torch.tensor([Tk, Tk - 30, 0], dtype=torch.int32)
    (q if where == "q" else go)[:, 3, 5] = bad
    got = _all(ops, q, k, v, go, H, 0.125, None, kv_lens, mask)
    keep = mask & (torch.arange(Tk)[None] < kv_lens[:, None])
    for n in ("dk", "dv"):
        assert (got[n].cpu()[~keep] == 0).all(), n
        clean = slice(d, None)          # the other head
        assert torch.isfinite(got[n][..., clean]).all(), n


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("Tk", [20, 100, 128, 129, 200])
def test_rows_without_keys_are_zero_whatever_they_hold(ops, Tk, bad):
    B, Tq, H, d = 3, 40, 2, 64
    q, k, v, go = _mk(B, Tq, Tk, H, H, d, torch.float16)
    mask = torch.rand(B, Tk, generator=torch.Generator().manual_seed(2)) < 0.7
    mask[1] = False
    kv_lens = torch.tensor([Tk, Tk, 0], dtype=torch.int32)
    q[1:, 3], go[1:, 4] = bad, bad
    want = _all(ops, q.nan_to_num(1.0, 1.0, 1.0), k, v, go.nan_to_num(1.0, 1.0, 1.0), H, 0.125, None, kv_lens, mask)
    for n, t in _all(ops, q, k, v, go, H, 0.125, None, kv_lens, mask).items():
        assert torch.equal(t[0], want[n][0]), n
        assert (t[1:] == (-math.inf if n == "lse" else 0)).all(), n


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("Tk,n", [(60, 33), (100, 64), (100, 70), (128, 65), (300, 128), (300, 200)])
def test_a_dropped_key_is_as_if_absent_also_for_values_that_are_not_finite(ops, Tk, n, bad):
    """Rows of q, k, v and go that are not finite give what the formula gives over the kept keys alone, whether others are masked, lie behind the length
    or are not stored at all: the same bits from the same kernel, NaN in the same places from another.  (Row 2's infinity meets one sign in every kept
    key: a score of +inf or -inf without a NaN of its own.)"""
    B, Tq, H, d = 4, 40, 1, 64
    q, k, v, go = _mk(B, Tq, Tk, H, H, d, torch.bfloat16)
    k[..., 7] = k[..., 7].abs() + 1
    q[:, 2, 7], q[1, 5], go[:, 9, 3] = bad, bad, bad
    k[2, 1, 0], v[3, 0, 0] = bad, bad
    lens, mask = torch.full((B,), n, dtype=torch.int32), torch.arange(Tk)[None].expand(B, -1) < n
    want = _all(ops, q, k[:, :n], v[:, :n], go, H, 0.125)
    for how in (dict(kv_lens=lens), dict(mask=mask)):
        got = _all(ops, q, k, v, go, H, 0.125, **how)
        for name in ("o", "lse", "dq"):
            if (n <= 128) == (Tk <= 128):
                _same(got[name], want[name], (name, tuple(how)))
            else:          # (two kernels, whose roundings differ)
                _same(got[name].float() * 0, want[name].float() * 0, (name, tuple(how)))


def _scaled(kind, B, Tq, Tk, H, d, dt):
    q, k, v, go = [t.float() for t in _mk(B, Tq, Tk, H, H, d, dt)]
    if kind == "large":               # states of thousands that line up with a small upstream gradient
        sign = torch.where(torch.rand(B, Tk, 1, generator=torch.Generator().manual_seed(Tk)) < 0.5, -1.0, 1.0)
        v, go = sign * (3000 + 100 * v), 1e-3 * (1 + go.abs())
    elif kind == "small":             # and small states
        q, k, v = q / 64, k * 64, v * 2.0 ** -10
    elif kind == "small_q":
        q, k, v = q * 64, k / 64, v * 2.0 ** -10
    elif kind == "rising":            # each tile's states larger than all before; the first ones are zero
        v = v * (torch.arange(Tk).float() / 8)[None, :, None] ** 2 / 4
        v[:, :5] = 0
    else:                             # falling
        v = v * 2000 / (1 + torch.arange(Tk).float())[None, :, None]
    return [t.to(dt) for t in (q, k, v, go)]


@pytest.mark.parametrize("kind", ["large", "small", "small_q", "rising", "falling"])
@pytest.mark.parametrize("Tq,Tk,d", [(5, 2, 64), (64, 77, 40), (40, 200, 64), (33, 300, 128), (2500, 70, 64), (130, 129, 160)])
def test_fp16_gradients_keep_their_range(ops, Tq, Tk, d, kind):
    """ds = p (go v - D) has the size of go v: an operand that only go's size places in fp16's range is infinite for large states, though every gradient is
    finite, and subnormal for small ones."""
    H = 2
    q, k, v, go = _scaled(kind, 2, Tq, Tk, H, d, torch.float16)
    R, E = _exact(q, k, v, go, H, d ** -0.5)
    assert all(float(R[n].abs().max()) < 6e4 for n in ("dq", "dk", "dv"))
    for n, t in _all(ops, q, k, v, go, H, d ** -0.5).items():
        _check(n, t, R, E)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Tq,Tk,H,G,d,kept", [(200, 129, 4, 4, 64, 2), (64, 300, 8, 2, 40, 3), (300, 1500, 4, 4, 64, 2), (100, 700, 4, 2, 128, 4), (100, 400, 2, 2, 160, 3),
                                              (100, 400, 2, 2, 24, 2), (90, 260, 2, 2, 96, 2)])
def test_few_kept_states_of_many_lose_only_the_roundings(ops, Tq, Tk, H, G, d, kept, dt):
    """The bar of few stored states (test_cross_attention_gpu) for few kept ones: two roundings, the ds operand's and the result's."""
    q, k, v, go = _mk(2, Tq, Tk, H, G, d, dt, Tk)
    mask = torch.zeros(2, Tk, dtype=torch.bool)
    for b in range(2):
        mask[b, torch.randperm(Tk, generator=torch.Generator().manual_seed(Tk + b))[:kept]] = True
    got = _all(ops, q, k, v, go, H, d ** -0.5, G, None, mask)
    R, E = _exact(q, k, v, go, H, d ** -0.5, G, None, mask)
    for n, t in got.items():
        _check(n, t, R, E)
    for n in ("dq", "dk"):
        assert float((got[n].double().cpu() - R[n]).norm() / R[n].norm()) <= 2 ** 0.5 * torch.finfo(dt).eps / (2 * 3 ** 0.5), n


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Tk,d", [(200, 64), (400, 40), (700, 128), (300, 160), (300, 96)])
def test_peaked_rows_of_many_states_lose_only_the_roundings(ops, Tk, d, dt):
    """Rows whose softmax is nearly one key: ds = p (dp - D) is small against D whatever the number of states."""
    H = 2
    q, k, v, go = _mk(2, 100, Tk, H, H, d, dt, Tk)
    q = (q.float() * 3).to(dt)
    got = _all(ops, q, k, v, go, H, d ** -0.5)
    R, E = _exact(q, k, v, go, H, d ** -0.5)
    for n, t in got.items():
        _check(n, t, R, E)
    for n in ("dq", "dk"):
        assert float((got[n].double().cpu() - R[n]).norm() / R[n].norm()) <= 2 ** 0.5 * torch.finfo(dt).eps / (2 * 3 ** 0.5), n


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Tq,Tk,H,G,d", [(1, 129, 1, 1, 8), (130, 200, 2, 2, 24), (33, 150, 4, 2, 32), (70, 260, 2, 1, 136), (140, 193, 2, 2, 160), (3, 640, 4, 1, 152)])
def test_tiled_kernels_at_the_ends_of_the_head_dims(ops, Tq, Tk, H, G, d, dt):
    """Over more than 128 states at the smallest and the largest head dims, with a mask and lengths that end inside a tile."""
    q, k, v, go = _mk(3, Tq, Tk, H, G, d, dt)
    lens = torch.tensor([Tk, Tk - 5, 1], dtype=torch.int32)
    mask = torch.rand(3, Tk, generator=torch.Generator().manual_seed(d)) < 0.8
    mask[2, 0] = True
    R, E = _exact(q, k, v, go, H, d ** -0.5, G, lens, mask)
    for n, t in _all(ops, q, k, v, go, H, d ** -0.5, G, lens, mask).items():
        _check(n, t, R, E)


@pytest.mark.parametrize("Tq,Tk", [(1, 32768), (200, 20000)])
def test_a_long_tail_of_small_probabilities_counts(ops, Tq, Tk):
    """One key holds nearly all of a row's weight and the others, each below fp16's smallest number beside it, hold 2^-10 of it together."""
    H, d = 2, 32
    q = torch.ones(1, Tq, H * d).half()
    k, v = torch.full((1, Tk, H * d), -17.5 / d).half(), torch.ones(1, Tk, H * d).half()
    k[0, 5], v[0, 5] = 0.0, 0.0
    v[0, :, ::3] = -2.0
    got = _all(ops, q, k, v, q, H, 1.0)
    R, E = _exact(q, k, v, q, H, 1.0)
    assert float(R["o"].abs().min()) > 2.0 ** -12
    for n in ("o", "lse"):
        _check(n, got[n], R, E)


@pytest.mark.parametrize("dt", TYPES)
def test_rows_too_far_apart_for_32_bit_offsets(ops, dt):
    """Few states under query, gradient and output rows 2^30 bytes apart: the kernels that address an item's rows with 32 bits leave them to the tiled ones."""
    B, Tq, Tk, H, d = 1, 3, 20, 2, 64
    q, k, v, go = _mk(B, Tq, Tk, H, H, d, dt)
    how = dict(q_lens=torch.tensor([3], dtype=torch.int32, device=DEV), kv_lens=torch.tensor([17], dtype=torch.int32, device=DEV))
    buf = torch.empty(2 * (1 << 29) + 4 * H * d, dtype=dt, device=DEV)

    def far(t, at):
        w = torch.as_strided(buf, t.shape, (3 << 29, 1 << 29, 1), at * H * d)
        w.copy_(t)
        return w
    (kd, vd), qd, gd = _fused_dev(k, v), far(q, 0), far(go, 1)
    o, lse = ops.cross_attention(qd, kd, vd, H, 0.125, want_lse=True, **how)
    got = dict(zip(("o", "lse", "dq", "dk", "dv"), (o, lse) + tuple(ops.cross_attention_bwd(qd, kd, vd, far(o, 2), lse, gd, H, 0.125, **how))))
    R, E = _exact(q, k, v, go, H, 0.125, None, torch.tensor([17]), None, late=True)
    for n, t in got.items():
        _check(n, t, R, E)


@pytest.mark.parametrize("Tk", [50, 200])
def test_queries_and_states_of_stride_zero(ops, Tk):
    """One query set for every item, one query row for every token, one state for every key."""
    B, Tq, H, d = 3, 20, 2, 64
    q, k, v, go = _dev(*_mk(B, Tq, Tk, H, H, d, torch.float16, fused=False))
    for qe, ke, ve in ((q[:1].expand(B, -1, -1), k, v), (q[:, :1].expand(-1, Tq, -1), k, v), (q, k[:, :1].expand(-1, Tk, -1), v[:, :1].expand(-1, Tk, -1))):
        want = ops.cross_attention(qe.contiguous(), ke.contiguous(), ve.contiguous(), H, 0.125, want_lse=True)
        got = ops.cross_attention(qe, ke, ve, H, 0.125, want_lse=True)
        grads = zip(ops.cross_attention_bwd(qe, ke, ve, *got, go[:, :1].expand(-1, Tq, -1), H, 0.125),
                    ops.cross_attention_bwd(qe.contiguous(), ke.contiguous(), ve.contiguous(), *want, go[:, :1].expand(-1, Tq, -1).contiguous(), H, 0.125))
        assert all(torch.equal(a, b) for a, b in list(zip(got, want)) + list(grads))


@pytest.mark.parametrize("Tk", [77, 150])
def test_more_than_2_to_the_31_outputs(ops, Tk):
    """The last item of a call whose queries, outputs and gradients pass 2^31 elements equals a call on that item alone."""
    B, Tq, H, d = 17, 65536, 16, 128
    g = torch.Generator(device=DEV).manual_seed(Tk)
    q = torch.empty(B, Tq, H * d, dtype=torch.bfloat16, device=DEV)
    q[:-1].fill_(0.25)
    q[-1].normal_(generator=g)
    kv = torch.randn(B, Tk, 2 * H * d, dtype=torch.bfloat16, device=DEV, generator=g)
    k, v = kv[..., :H * d], kv[..., H * d:]
    assert q.numel() > 1 << 31
    o, lse = ops.cross_attention(q, k, v, H, 0.1, want_lse=True)
    dq, dk, dv = ops.cross_attention_bwd(q, k, v, o, lse, q, H, 0.1)
    o1, lse1 = ops.cross_attention(q[-1:], k[-1:], v[-1:], H, 0.1, want_lse=True)
    dq1, dk1, dv1 = ops.cross_attention_bwd(q[-1:], k[-1:], v[-1:], o1, lse1, q[-1:], H, 0.1)
    assert torch.equal(o[-1:], o1) and torch.equal(lse[-1:], lse1) and torch.equal(dq[-1:], dq1)
    for a, b in ((dk, dk1), (dv, dv1)):          # (alone, the rows are cut into other slices: the same but for the order of fp32 sums and one rounding)
        assert float((a[-1:].double() - b.double()).norm() / b.double().norm()) <= torch.finfo(torch.bfloat16).eps / 2


def test_two_threads_at_once(ops):
    """Calls from two host threads, each on a stream of its own, give what they give one after the other."""
    import threading
    sets = [_dev(*_mk(2, 300 + 50 * i, 70 + 100 * i, 4, 2, 64, torch.float16, seed=i, fused=False)) for i in range(2)]
    pws = [ops.pack_w_fp8(torch.randn(512 + 64 * i, 256, generator=torch.Generator().manual_seed(i)).to(DEV)) for i in range(2)]

    def one(i):
        q, k, v, go = sets[i]
        o, lse = ops.cross_attention(q, k, v, 4, 0.125, 2, want_lse=True)
        y = ops.linear_fp8(o, pws[i])
        return (o, lse, y) + tuple(ops.cross_attention_bwd(q, k, v, o, lse, go, 4, 0.125, 2)) + tuple(ops.linear_fp8_bwd(o, y, pws[i]))
    want = [one(0), one(1)]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got[i] = one(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:          # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])), i


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Tk,kept", [(16, 16), (100, 20), (200, 16), (300, 300)])
def test_far_scores_do_not_unbalance_the_gradients(ops, Tk, kept, dt):
    """Scores near +-100, rows whose softmax is nearly one key.  Recomputed probabilities sum to one only up to the rounding of lse, some 2^-23 |lse|, and that
    times D is not small against ds = p (dp - D).  All inputs are small integers: scores and dp are exact, a probability is off by
    e = 2^-21 + 3 2^-24 max|score| relative to the row's others and in common, so ds before its rounding by at most e (|ds| + p sum |ds|) and by the fp32
    sum D, (n + 4) 2^-24 p (|dp| + sum p |dp|)."""
    B, Tq, H, d = 1, 64, 1, 32
    u, half = torch.finfo(dt).eps / 2, dt == torch.float16
    g = torch.Generator().manual_seed(Tk)
    q, k, v, go = (torch.zeros(B, T, d) for T in (Tq, Tk, Tk, Tq))
    q[:, ::2, 0], q[:, 1::2, 0] = 1, -1
    k[0, :, 0] = torch.randint(80, 94, (Tk,), generator=g).float()
    mask = torch.zeros(B, Tk, dtype=torch.bool)
    mask[0, torch.randperm(Tk, generator=g)[:kept]] = True
    idx = mask[0].nonzero()[:, 0]
    k[0, idx[0], 0], k[0, idx[1], 0] = 102, 72
    k[..., 1:] = torch.randint(-2, 3, k[..., 1:].shape, generator=g).float()
    v[:] = 8 + torch.randint(-3, 4, v.shape, generator=g).float()
    go[:] = 2 + torch.randint(-2, 3, go.shape, generator=g).float()
    q, k, v, go = (t.to(dt) for t in (q, k, v, go))
    got = _all(ops, q, k, v, go, H, 1.0, None, None, mask)
    R, _ = _exact(q, k, v, go, H, 1.0, None, None, mask)
    qq, kk, vv, gg = (t[0].double() for t in (q, k[:, idx], v[:, idx], go))
    s, dp = qq @ kk.t(), gg @ vv.t()
    p = torch.softmax(s, -1)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    e = 2.0 ** -21 + 3 * 2.0 ** -24 * float(s.abs().max())
    und = 2.0 ** -33 * (dp - (p * dp).sum(-1, keepdim=True)).abs().amax() if half else 2.0 ** -126
    A = (p * dp.abs()).sum(-1, keepdim=True)
    # over many states D starts from the rounded o: the correction is itself rounded twice
    more = 2 * u * u * (p @ vv.abs() * gg.abs()).sum(-1, keepdim=True) * p if Tk > 128 else 0.0
    Ed = u * ds.abs() + e * (ds.abs() + p * ds.abs().sum(-1, keepdim=True)) + (kept + 4) * 2.0 ** -24 * p * (dp.abs() + A) + und + more
    tiny = 2.0 ** -25 if half else 2.0 ** -126
    E = {"dq": torch.zeros_like(R["dq"]), "dk": torch.zeros_like(R["dk"])}
    E["dq"][0] = (Ed + kept * 2.0 ** -24 * ds.abs()) @ kk.abs() + u * R["dq"][0].abs() + tiny
    E["dk"][0, idx] = (Ed + Tq * 2.0 ** -24 * ds.abs()).t() @ qq.abs() + u * R["dk"][0, idx].abs() + tiny
    for n in E:
        _check(n, got[n], R, E)


@pytest.mark.parametrize("dt", TYPES)
def test_a_million_states(ops, dt):
    Tk, H, d = (1 << 20) + 77, 1, 32
    q, k, v, go = _mk(1, 2, Tk, H, H, d, dt)
    lens = torch.tensor([Tk - 100], dtype=torch.int32)
    R, E = _exact(q, k, v, go, H, d ** -0.5, None, lens)
    for n, t in _all(ops, q, k, v, go, H, d ** -0.5, None, lens).items():
        _check(n, t, R, E)


def test_more_items_than_a_launch_holds_are_refused(ops):
    """2^24 pairs of item and key head (one query each, every item reading the same rows): refused on the host, nothing launched; half of them run."""
    B, d = 1 << 18, 8
    for H in (32, 64):
        q, k = (torch.ones(1, T, H * d, dtype=torch.float16, device=DEV).expand(B, -1, -1) for T in (1, 2))
        if H == 32:
            assert (ops.cross_attention(q, k, k, H, 0.5) == 1).all()
            continue
        with pytest.raises(ops.TfmqError, match="too many workgroups"):
            ops.cross_attention(q, k, k, H, 0.5)
        with pytest.raises(ops.TfmqError, match="too many workgroups"):
            ops.cross_attention_bwd(q, k, k, q, torch.zeros(B, H, 1, device=DEV), q, H, 0.5)
