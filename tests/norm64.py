"""Layer norm and its gradients in 64 bits, with how far fp32 sums may be from them.

A device sum is a chain of at most 64 additions in a lane, 6 steps over the wave and up to 4 over the block's waves: each rounds by 2^-24 of
a partial sum, so a sum of D values is off by at most 80 * 2^-24 of the sum of their magnitudes. That goes for the mean (`dm`, which
moves every normed value of the row by dm r), the variance (half of its relative error for r) and the means of g and g n. Sums over
rows are chains of at most 64 rows of a wave, 4 waves and 2 * 32 blocks: 160 * 2^-24 of the sum of magnitudes, beside the errors of the normed
values in them. The few products around them are counted by rounding the factors up."""
import torch

U = 2.0 ** -24
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}   # half a subnormal step


def stats(x, eps):
    """n, r and the error of n."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    r = (c.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    n = c * r
    dm = 84 * U * x.abs().mean(-1, keepdim=True)
    return n, r, dm * r + (50 * U + (dm * r).pow(2)) * n.abs() + U * x.abs() * r


def norm(x, w, b, eps):
    n, _, en = stats(x, eps)
    w = 1.0 if w is None else w.double()
    y, err = n * w, en * (abs(w) if isinstance(w, float) else w.abs())
    if b is not None:
        y = y + b.double()
    return y, err + 3 * U * ((n * w).abs() + y.abs())


def backward(dy, x, gain, eps, rows_dim=0):
    """(dx, its error), (sum dy n, its error), (sum dy, its error); gain broadcasts against x, sums are over rows_dim."""
    n, r, en = stats(x, eps)
    dy = dy.double()
    g = dy * gain
    mg, mgn = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    ag, agn = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    emgn = 90 * U * agn + (g.abs() * en).mean(-1, keepdim=True)
    dx = r * (g - mg - n * mgn)
    edx = r * (4 * U * g.abs() + 84 * U * ag + en * mgn.abs() + n.abs() * (emgn + 4 * U * mgn.abs())) + 50 * U * dx.abs()
    ew = 164 * U * (dy * n).abs().sum(rows_dim) + (dy.abs() * en).sum(rows_dim)
    return (dx, edx), ((dy * n).sum(rows_dim), ew), (dy.sum(rows_dim), 164 * U * dy.abs().sum(rows_dim))


def close(got, want, err, what=""):
    """got within half a step of its type and err (that of the value rounded) of want."""
    want, err = want.to(got.device), err.to(got.device)
    room = (want.abs() + err) * STEP[got.dtype] + err + TINY[got.dtype]
    off = (got.double() - want).abs()
    ok = (off <= room).all()
    assert ok, f"{what}: off by {float((off / room).max()):.3g} of what is allowed at {int((off / room).argmax())}"
