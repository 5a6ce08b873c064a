"""Adapters of many requests and their gradients in 64 bits, with how far the device's sums may be from them.

A product of two 16-bit values is exact in fp32; the matrix cores add 32 of them in an instruction and instructions add up in a chain, each addition cut or
rounded: 2^-23 of a partial sum. A sum of K products (K / 32 instructions, 32 in the last, 4 waves, 16 slices) is off by at most
(K / 32 + 64) 2^-23 of the sum of magnitudes. Narrow values enter the second product as two bf16: 2^-16 of the value is left out, and as much
once more where they meet fp16 (its second part times theirs); their scale rounds by 2^-24. A sum over T rows is up to 3 T / 32
additions, 32 within an instruction and 64 parts."""
import torch

U23 = 2.0 ** -23


def left_out(dtype):
    return 2.0 ** -16 * (2 if dtype == torch.float16 else 1) + 2.0 ** -24


def narrow(x, w):
    """x w^T and its error: x [T, K], w [R, K]."""
    return x @ w.t(), (x.abs() @ w.abs().t()) * (x.shape[1] / 32 + 64) * U23


def wide(h, eh, f, w, dtype):
    """f h w^T: h [T, R], w [C, R]."""
    R = h.shape[1]
    y = f * (h @ w.t())
    return y, f.abs() * ((h.abs() * (left_out(dtype) + (3 * R / 32 + 40) * U23) + eh) @ w.abs().t())


def outer(q, eq, f, v, dtype):
    """f q^T v over rows: q [T, R], v [T, C]."""
    T = q.shape[0]
    room = left_out(dtype) + (3 * T / 32 + 100) * U23
    return f * (q.t() @ v), f.abs() * ((q.abs() * room + eq).t() @ v.abs())


def forward(base, x, a, b, scale, index):
    """(out, err) for 2-D base and x."""
    per = x.shape[0] // index.numel() if index.numel() else 0
    of = index.reshape(-1).long().repeat_interleave(per) if per else index.long()
    out, err = base.double(), torch.zeros_like(base, dtype=torch.float64)
    for i in range(a.shape[0]):
        t = (of == i).nonzero()[:, 0]
        if len(t):
            h, eh = narrow(x[t].double(), a[i].double())
            y, ey = wide(h, eh, scale[i].double(), b[i].double(), x.dtype)
            out[t] += y
            err[t] = ey + out[t].abs() * 2.0 ** -24
    return out, err


def backward(dy, x, a, b, scale, index):
    """((dx, err), (da, err), (db, err)) for 2-D dy and x."""
    per = x.shape[0] // index.numel() if index.numel() else 0
    of = index.reshape(-1).long().repeat_interleave(per) if per else index.long()
    zeros = [(torch.zeros(s.shape, dtype=torch.float64, device=x.device), torch.zeros(s.shape, dtype=torch.float64, device=x.device)) for s in (x, a, b)]
    (dx, ex), (da, ea), (db, eb) = zeros
    for i in range(a.shape[0]):
        t = (of == i).nonzero()[:, 0]
        if len(t) == 0:
            continue
        xi, yi, ai, bi, f = x[t].double(), dy[t].double(), a[i].double(), b[i].double(), scale[i].double()
        h, eh = narrow(xi, ai)
        g, eg = narrow(yi, bi.t().contiguous())
        dx[t], ex[t] = wide(g, eg, f, ai.t().contiguous(), x.dtype)
        da[i], ea[i] = outer(g, eg, f, xi, x.dtype)
        d, e = outer(h, eh, f, yi, x.dtype)
        db[i], eb[i] = d.t(), e.t()
    return zeros
