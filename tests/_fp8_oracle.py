"""64-bit oracle of the e4m3 block quantisation: written from the definition, on the CPU."""
import torch

F8_MAX, AMAX_MIN = 448.0, 2.0 ** -100


def e4m3(v):
    """Nearest e4m3 value (ties to even) of float64 values of magnitude <= 448 (1 + 2^-20); NaN stays."""
    _, ex = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (ex - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def scales(a):
    """a float64 >= 0 -> (reciprocal, scale), the fp32 numbers as float64."""
    a = torch.where(torch.isnan(a), a, torch.maximum(a, torch.full_like(a, AMAX_MIN)))
    return (F8_MAX / a).float().double(), (a / F8_MAX).float().double()


def quant(x, rows=1):
    """[R, K] -> (q values float64 [R, K], scales float64 [R, Kb]) with one scale per `rows` x 128 block (given per row)."""
    x = x.detach().cpu().double()
    R, K = x.shape
    Kb = (K + 127) // 128
    q, s = torch.empty_like(x), torch.empty(R, Kb, dtype=torch.float64)
    for b in range(Kb):
        blk = x[:, b * 128:(b + 1) * 128]
        for r0 in range(0, R, rows):
            part = blk[r0:r0 + rows]
            a = part.abs().amax(1, keepdim=True) if rows == 1 else part.abs().max().reshape(1, 1)
            r, sc = scales(a)
            q[r0:r0 + rows, b * 128:(b + 1) * 128] = e4m3((part * r).float().double())
            s[r0:r0 + rows, b] = sc[:, 0]
    return q, s


def quant_rows(x):
    """quant(x, 1) without the Python loop over rows."""
    x = x.detach().cpu().double()
    R, K = x.shape
    Kb = (K + 127) // 128
    q, s = torch.empty_like(x), torch.empty(R, Kb, dtype=torch.float64)
    for b in range(Kb):
        blk = x[:, b * 128:(b + 1) * 128]
        r, sc = scales(blk.abs().amax(1, keepdim=True))
        q[:, b * 128:(b + 1) * 128] = e4m3((blk * r).float().double())
        s[:, b] = sc[:, 0]
    return q, s


def dequant(q, s):
    return q * s.repeat_interleave(128, 1)[:, :q.shape[1]]
