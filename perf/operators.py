"""The measured cases of the 8-bit float Linear and of the cross attention to an encoder's states.

Two families: a Linear on e4m3 operands with one scale per block of 128 (forward, and its gradients), and the attention of B x Tq query tokens to
Tk states of an encoder, with per-item lengths, a key mask and shared key / value heads (forward, and a training pass).  `own` selects the
framework's entry points; otherwise `run` computes the plain form from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

F8_MAX = 448.0
AMAX_MIN = 2.0 ** -100
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------------- cases
def _lin(name, M, K, N, t, bias=True):
    return {"name": name, "op": "linear", "M": M, "K": K, "N": N, "t": t, "bias": bias}


def _linb(name, M, K, N, t):
    return {"name": name, "op": "linear_bwd", "M": M, "K": K, "N": N, "t": t}


def _att(name, op, B, Tq, Tk, heads, kv_heads, d, t, lens, mask):
    return {"name": name, "op": op, "B": B, "Tq": Tq, "Tk": Tk, "heads": heads, "kv_heads": kv_heads, "d": d, "t": t, "lens": lens, "mask": mask}


def listed():
    return [
        # the time-embedding Linear of one image under guidance: two rows, a call of latency
        _lin("linear_2rows", 2, 1280, 1280, "f16"),
        # the fused k | v projection of two prompts of 77 tokens
        _lin("linear_context", 154, 768, 1280, "bf16", bias=False),
        # the gated feed-forward's first projection at the 64 x 64 level of two images: K is two and a half blocks
        _lin("linear_ff_64", 8192, 320, 2560, "f16"),
        # the same projection at the 16 x 16 level of 64 images: the largest product
        _lin("linear_ff_16", 16384, 1280, 10240, "f16"),
        # gradients of a square token Linear over eight images of the 32 x 32 level
        _linb("linear_bwd_tokens", 8192, 640, 640, "bf16"),
        # gradients over a ragged token count and odd widths
        _linb("linear_bwd_odd", 1333, 1000, 777, "f16"),
        # the 64 x 64 level of one image under guidance, prompts of different lengths
        _att("cross_pair_64", "cross", 2, 4096, 77, 8, 8, 40, "f16", True, False),
        # the 32 x 32 level of 64 images under guidance, masked prompt tokens
        _att("cross_batch_32", "cross", 128, 1024, 77, 8, 8, 80, "bf16", False, True),
        # one new token for each of 16 sequences against long states, four query heads to a key head
        _att("cross_one_token", "cross", 16, 1, 4095, 32, 8, 128, "bf16", True, False),
        # long queries to long states
        _att("cross_long", "cross", 2, 4096, 4096, 16, 16, 64, "f16", True, False),
        # a training pass of the 64 x 64 level at the recipe's mini-batch of eight
        _att("cross_train_64", "cross_train", 8, 4096, 77, 8, 8, 40, "f16", True, False),
        # a training pass over longer, ragged states with shared key heads
        _att("cross_train_long", "cross_train", 4, 1000, 1500, 16, 4, 128, "bf16", True, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_bwd", "cross", "cross", "cross_train"])
    most = max(work(c)["flops"] for c in listed() if c["op"] == op)
    while True:
        t = rng.choice(["f16", "bf16"])
        if op in ("linear", "linear_bwd"):
            if op == "linear" and rng.random() < 0.2:
                t = "f32"
            c = {"op": op, "M": _log_int(rng, 1, 16384), "K": _log_int(rng, 64, 5120), "N": _log_int(rng, 64, 10240), "t": t}
            if rng.random() < 0.5:          # widths of models are mostly multiples of 64
                c["K"], c["N"] = (c["K"] + 63) // 64 * 64, (c["N"] + 63) // 64 * 64
            if op == "linear":
                c["bias"] = rng.random() < 0.5
        else:
            heads = rng.choice([4, 5, 8, 16, 32])
            kv = rng.choice([g for g in (1, heads // 4, heads // 2, heads, heads, heads) if g >= 1 and heads % g == 0])
            # (a gradient through a single state is zero, and says nothing: training draws start at sixteen)
            tq = 1 if (op == "cross" and rng.random() < 0.3) else _log_int(rng, 2, 4096)
            c = {"op": op, "B": _log_int(rng, 1, 64), "Tq": tq, "Tk": _log_int(rng, 16 if op == "cross_train" else 1, 4096), "heads": heads, "kv_heads": kv,
                 "d": rng.choice([32, 40, 64, 80, 96, 128, 160]), "t": t, "lens": rng.random() < 0.6, "mask": rng.random() < 0.4}
            if c["B"] * heads * tq * c["Tk"] > 600e6 or c["B"] * c["Tk"] * kv * c["d"] > 3e8:
                continue
        if work(c)["flops"] <= most:
            return c


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed, *parts):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + sum((i + 1) * int(p) for i, p in enumerate(parts))) % (2 ** 62))
    return g


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    dt = TYPES[case["t"]]
    dev = "cuda"
    if case["op"] in ("linear", "linear_bwd"):
        M, K, N = case["M"], case["K"], case["N"]
        g = _gen(seed, M, K, N)
        # activations behind a norm: unit variance with a few channels that stand out, as token streams have them
        x = torch.randn(M, K, generator=g, device=dev)
        gain = 1.0 + 7.0 * (torch.rand(K, generator=g, device=dev) < 0.02).float()
        w = torch.randn(N, K, generator=g, device=dev) * K ** -0.5
        s = {"x": (x * gain).to(dt), "w": w}
        if case["op"] == "linear":
            s["bias"] = torch.randn(N, generator=g, device=dev) * 0.1 if case["bias"] else None
        else:
            s["gy"] = (torch.randn(M, N, generator=g, device=dev) * torch.rand(M, 1, generator=g, device=dev)).to(dt)
        return s
    B, Tq, Tk, H, G, d = (case[k] for k in ("B", "Tq", "Tk", "heads", "kv_heads", "d"))
    g = _gen(seed, B, Tq, Tk, H, G, d)
    s = {"q": torch.randn(B, Tq, H * d, generator=g, device=dev).to(dt)}
    # k and v as the two halves of one fused projection's rows
    kv = torch.randn(B, Tk, 2 * G * d, generator=g, device=dev).to(dt)
    s["k"], s["v"] = kv[..., :G * d], kv[..., G * d:]
    s["lens"] = torch.randint(max(1, Tk // 4), Tk + 1, (B,), generator=g, device=dev, dtype=torch.int32) if case["lens"] else None
    s["mask"] = (torch.rand(B, Tk, generator=g, device=dev) < 0.8) if case["mask"] else None
    if s["lens"] is not None and B > 2:
        s["lens"][B // 2] = 0               # an item without states: its rows are zero
    s["scale"] = d ** -0.5
    if case["op"] == "cross_train":
        s["go"] = torch.randn(B, Tq, H * d, generator=g, device=dev).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    if case["op"] in ("linear", "linear_bwd"):
        # a program quantises its weights once and keeps them
        if own:
            import tfmq_dm_amd.ops as ops
            s["ops"] = ops
            s["pw"] = ops.pack_w_fp8(s.pop("w"), s.get("bias"))
        else:
            s["wq"] = _quant_weight(s.pop("w"))
    elif own:
        import tfmq_dm_amd.ops as ops
        s["ops"] = ops
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _scales(a):
    """Reciprocal and scale of blocks whose largest magnitude is a: the 32-bit numbers next to 448 / a and a / 448.  Taken in 64 bits: values
    of 16-bit types often fall on the border between two e4m3 values exactly, and a last bit of the reciprocal decides there."""
    a = a.double().clamp_min(AMAX_MIN)
    return (F8_MAX / a).float(), (a / F8_MAX).float()


def _quant_rows(x):
    """Values of x [R, K] in e4m3 with a scale per row and block of 128 columns: back in 32 bits, scale applied."""
    R, K = x.shape
    nb = (K + 127) // 128
    xp = torch.zeros(R, nb * 128, dtype=torch.float32, device=x.device)
    xp[:, :K] = x.float()
    xb = xp.view(R, nb, 128)
    r, sc = _scales(xb.abs().amax(-1, keepdim=True))
    q = (xb * r).to(torch.float8_e4m3fn).float()
    return (q * sc).view(R, nb * 128)[:, :K]


def _quant_weight(w):
    """The same with a scale per block of 128 x 128."""
    N, K = w.shape
    nn, nk = (N + 127) // 128, (K + 127) // 128
    wp = torch.zeros(nn * 128, nk * 128, dtype=torch.float32, device=w.device)
    wp[:N, :K] = w.float()
    wb = wp.view(nn, 128, nk, 128)
    r, sc = _scales(wb.abs().amax((1, 3), keepdim=True))
    q = (wb * r).to(torch.float8_e4m3fn).float()
    return (q * sc).view(nn * 128, nk * 128)[:N, :K].contiguous()


def _keep(s, B, Tk):
    keep = torch.ones(B, Tk, dtype=torch.bool, device=s["q"].device)
    if s["lens"] is not None:
        keep &= torch.arange(Tk, device=keep.device)[None, :] < s["lens"][:, None]
    if s["mask"] is not None:
        keep &= s["mask"]
    return keep


def _heads(x, n, rep, dt=torch.float32):
    """[B, T, n * d] -> [B, n * rep, T, d], each head repeated for the query heads that share it."""
    B, T, C = x.shape
    y = x.to(dt).reshape(B, T, n, C // n).permute(0, 2, 1, 3).contiguous()
    return y.repeat_interleave(rep, dim=1) if rep > 1 else y


def _rows(x, dt):
    B, H, T, d = x.shape
    return x.permute(0, 2, 1, 3).reshape(B, T, H * d).to(dt)


def _attend(s, case):
    H, G = case["heads"], case["kv_heads"]
    q, k, v = _heads(s["q"], H, 1), _heads(s["k"], G, H // G), _heads(s["v"], G, H // G)
    keep = _keep(s, case["B"], case["Tk"])[:, None, None, :]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    x = torch.where(keep, x, torch.full_like(x, -math.inf))
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    return q, k, v, p, torch.matmul(p, v)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "linear":
        y = torch.matmul(_quant_rows(s["x"]), s["wq"].t())
        if s["bias"] is not None:
            y = y + s["bias"]
        return y.to(s["x"].dtype)
    if op == "linear_bwd":
        gx = torch.matmul(_quant_rows(s["gy"]), s["wq"]).to(s["x"].dtype)
        gw = torch.matmul(_quant_rows(s["gy"].t()), _quant_rows(s["x"].t()).t())
        return gx, gw
    dt = s["q"].dtype
    q, k, v, p, o = _attend(s, case)
    if op == "cross":
        return _rows(o, dt)
    B, H, G, d = case["B"], case["heads"], case["kv_heads"], case["d"]
    go = _heads(s["go"], H, 1)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), go)
    dp = torch.matmul(go, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (o * go).sum(-1, keepdim=True)) * s["scale"]
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    if H != G:
        dk, dv = (t.view(B, G, H // G, case["Tk"], d).sum(2) for t in (dk, dv))
    return _rows(o, dt), _rows(dq, dt), _rows(dk, dt), _rows(dv, dt)


def run(state):
    if not own:
        return _plain(state)
    s, ops = state, state["ops"]
    case = s["case"]
    op = case["op"]
    if op == "linear":
        return ops.linear_fp8(s["x"], s["pw"])
    if op == "linear_bwd":
        return ops.linear_fp8_bwd(s["x"], s["gy"], s["pw"])
    how = dict(kv_heads=case["kv_heads"], kv_lens=s["lens"], mask=s["mask"])
    if op == "cross":
        return ops.cross_attention(s["q"], s["k"], s["v"], case["heads"], s["scale"], **how)
    o, lse = ops.cross_attention(s["q"], s["k"], s["v"], case["heads"], s["scale"], want_lse=True, **how)
    return (o,) + tuple(ops.cross_attention_bwd(s["q"], s["k"], s["v"], o, lse, s["go"], case["heads"], s["scale"], **how))


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    e = SIZE[case["t"]]
    if case["op"] in ("linear", "linear_bwd"):
        M, K, N = case["M"], case["K"], case["N"]
        w = N * K + 4 * ((N + 127) // 128) * ((K + 127) // 128)
        if case["op"] == "linear":
            return {"bytes": e * M * (K + N) + w + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
        return {"bytes": e * M * (2 * K + N) + w + 4 * N * K, "flops": 4 * M * N * K}
    B, Tq, Tk, H, G, d = (case[k] for k in ("B", "Tq", "Tk", "heads", "kv_heads", "d"))
    side = (4 * B if case["lens"] else 0) + (B * Tk if case["mask"] else 0)
    share = 0.625 if case["lens"] else 1.0          # the mean length over the stored one: keys behind it are neither read nor multiplied
    if case["op"] == "cross":
        return {"bytes": int(e * B * d * (2 * Tq * H + 2 * share * Tk * G)) + side, "flops": int(4 * share * B * H * Tq * Tk * d)}
    return {"bytes": int(e * B * d * (4 * Tq * H + 2 * (share + 1) * Tk * G)) + side, "flops": int(14 * share * B * H * Tq * Tk * d)}


# ----------------------------------------------------------------------------------------------------------------- exact
def _e4m3(v):
    """Nearest e4m3 value, ties to even, of float64 values within the type's range."""
    _, ex = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (ex - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _exact_rows(x, rows):
    """The 64-bit values of x quantised with one scale per `rows` x 128 block; scale and reciprocal are 32-bit numbers by definition."""
    x = x.double()
    out = torch.empty_like(x)
    R, K = x.shape
    for c in range(0, K, 128):
        blk = x[:, c:c + 128]
        a = blk.abs().amax(1)
        if rows > 1:
            a = torch.cat([a[i:i + rows].max().expand(min(rows, R - i)) for i in range(0, R, rows)])
        a = torch.maximum(a, torch.full_like(a, AMAX_MIN))[:, None]
        r, sc = (F8_MAX / a).float().double(), (a / F8_MAX).float().double()
        out[:, c:c + 128] = _e4m3((blk * r).float().double()) * sc
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("linear", "linear_bwd"):
        w = _exact_rows(s["w"], 128)
        if op == "linear":
            y = _exact_rows(s["x"], 1) @ w.t()
            return y if s["bias"] is None else y + s["bias"].double()
        gy, x = s["gy"], s["x"]
        return _exact_rows(gy, 1) @ w, _exact_rows(gy.t().contiguous(), 1) @ _exact_rows(x.t().contiguous(), 1).t()
    B, Tq, Tk, H, G, d = (case[k] for k in ("B", "Tq", "Tk", "heads", "kv_heads", "d"))
    outs = [torch.zeros_like(s["q"], dtype=torch.float64)]
    if op == "cross_train":
        outs += [torch.zeros_like(s["q"], dtype=torch.float64)] + [torch.zeros(B, Tk, G * d, dtype=torch.float64, device="cuda") for _ in range(2)]
    for b in range(B):
        idx = torch.arange(Tk, device="cuda")
        if s["lens"] is not None:
            idx = idx[idx < s["lens"][b]]
        if s["mask"] is not None:
            idx = idx[s["mask"][b][idx]]
        if idx.numel() == 0:
            continue
        for h in range(H):
            cq, ck = slice(h * d, (h + 1) * d), slice((h // (H // G)) * d, (h // (H // G) + 1) * d)
            q, k, v = s["q"][b, :, cq].double(), s["k"][b, idx, ck].double(), s["v"][b, idx, ck].double()
            p = torch.softmax(q @ k.t() * s["scale"], -1)
            o = p @ v
            outs[0][b, :, cq] = o
            if op == "cross_train":
                go = s["go"][b, :, cq].double()
                ds = p * (go @ v.t() - (o * go).sum(-1, keepdim=True)) * s["scale"]
                outs[1][b, :, cq] = ds @ k
                outs[2][b, idx, ck] += ds.t() @ q
                outs[3][b, idx, ck] += p.t() @ go
    return outs[0] if op == "cross" else tuple(outs)
