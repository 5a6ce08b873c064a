"""The router's scores, balance loss and gradients in 64 bits, with how far the device may be from them.

A logit is a sum of D exact products: off by (D / 32 + 64) 2^-23 of their magnitudes (see adapters64). A score moves by the errors of its own logit and of
those in its sum, relative to itself, and by the exponential, the sum and the division: 8 * 2^-23. A mean of scores adds tiles of 64 in at most 64
+ 32 + 64 steps (T up to 2^18 here): 200 * 2^-24. dz has a few roundings (8 * 2^-24) of dp and of the sum of p dp beside the scores' errors, and
enters its two products as adapters64's narrow values do."""
import torch

from tests.adapters64 import U23, left_out

U = 2.0 ** -24


def balance(x, w, idx, alpha, sequences, mask, dloss=None, dweight=None):
    """(loss, err), counts, (scores, err) and, with dloss, (dx, err), (dW, err)."""
    T, D = x.shape
    E, k = w.shape[0], idx.shape[1]
    L = T // sequences
    x64, w64 = x.double(), w.double()
    keep = torch.ones(T, dtype=torch.bool, device=x.device) if mask is None else mask.reshape(-1)
    p = torch.softmax(x64 @ w64.t(), 1)
    ez = (x64.abs() @ w64.abs().t()) * (D / 32 + 64) * U23
    ep = p * (ez + (p * ez).sum(1, keepdim=True) + 8 * U23) * 1.01
    one = (idx.long()[:, :, None] == torch.arange(E, device=x.device)) & keep[:, None, None]
    counts = one.view(sequences, L * k, E).sum(1)
    n = keep.view(sequences, L).sum(1)
    held = max(1, int((n > 0).sum()))
    full = torch.where(n > 0, 1.0 / n.clamp_min(1).double(), 0.0)[:, None]
    load = E * counts.double() * full / k
    pk, ek = (torch.where(keep[:, None], v, 0.0).view(sequences, L, E).sum(1) * full for v in (p, ep))
    loss = alpha * (load * pk).sum() / held
    eloss = abs(alpha) * (load * (ek + 220 * U * pk)).sum() / held
    if dloss is None:
        return (loss, eloss), counts, (p, ep)
    dp = (dloss.double() * alpha / held * load * full)[:, None].expand(sequences, L, E).reshape(T, E).clone()
    mag = dp.abs()
    if dweight is not None:
        for j in range(k):
            add = one[:, j].double() * dweight[:, j:j + 1].double()
            dp, mag = dp + add, mag + add.abs()
    dot = (p * dp).sum(1, keepdim=True)
    edot = (ep * mag + 12 * U * p * mag).sum(1, keepdim=True)
    keep = keep[:, None]
    dz = torch.where(keep, p * (dp - dot), 0.0)
    edz = torch.where(keep, ep * (dp - dot).abs() + p * (8 * U * mag + edot) + 4 * U * dz.abs(), 0.0)
    room = left_out(x.dtype)
    dx = dz @ w64
    edx = (dz.abs() * (room + 40 * U23) + edz) @ w64.abs()
    xk = torch.where(keep, x64, 0.0)
    dw = dz.t() @ xk
    edw = (dz.abs() * (room + (3 * T / 32 + 100) * U23) + edz).t() @ xk.abs()
    return (loss, eloss), counts, (p, ep), (dx, edx), (dw, edw)
