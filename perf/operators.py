"""Measured cases of the fp8 operators with a scale for each block of 128: the cast of 16-bit rows, the Linear, the Linears of
experts over ragged row segments, and the experts' SwiGLU feed-forward.

  cast      s = max(max|x|, 2^-96) / 448 of every 128 values of a row, q = e4m3fn(x * (448 / max(max|x|, 2^-96)))
  linear    y = (q s) (w sw)^T + bias, sw one value for each 128 x 128 block of w, y rounded once
  grouped   the same for the rows [offsets[e], offsets[e + 1]) with expert e's weight
  ffn       y = cast(silu(x w1^T) * (x w3^T)) w2^T for every expert's rows, x cast before

`own` chooses between the plain form of an operator and this package's."""
import math

import torch

own = False

BLOCK = 128
FLOOR = 2.0 ** -96
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # activations of a short prompt in front of one Linear; the tokens of a large batch
        {"name": "cast 333 rows", "op": "cast", "rows": 333, "K": 2560, "dtype": "bf16"},
        {"name": "cast 32768 rows", "op": "cast", "rows": 32768, "K": 6912, "dtype": "bf16"},
        # one token, a few tokens, a 3-D shape's tokens with a bias, a large batch
        {"name": "linear 1 row", "op": "linear", "rows": 1, "K": 2560, "N": 6912, "dtype": "bf16", "bias": False},
        {"name": "linear 48 rows", "op": "linear", "rows": 48, "K": 6912, "N": 2560, "dtype": "fp16", "bias": True},
        {"name": "linear 1500 rows", "op": "linear", "rows": 1500, "K": 2048, "N": 8192, "dtype": "fp16", "bias": True},
        {"name": "linear 16384 rows", "op": "linear", "rows": 16384, "K": 4096, "N": 8192, "dtype": "bf16", "bias": False},
        # the down projection of a few tokens of a top-2 layer; experts of another size, one of them without rows; a large batch
        {"name": "grouped 128 rows", "op": "grouped", "rows": 128, "K": 6912, "N": 2560, "E": 4, "empty": 0, "dtype": "bf16"},
        {"name": "grouped 3001 rows", "op": "grouped", "rows": 3001, "K": 2048, "N": 8192, "E": 8, "empty": 1, "dtype": "fp16"},
        {"name": "grouped 16384 rows", "op": "grouped", "rows": 16384, "K": 6912, "N": 2560, "E": 4, "empty": 0, "dtype": "bf16"},
        # one token of a top-2 layer, a small image, a large one
        {"name": "ffn 2 rows", "op": "ffn", "rows": 2, "K": 2560, "H": 6912, "E": 4, "empty": 0, "dtype": "bf16"},
        {"name": "ffn 1021 rows", "op": "ffn", "rows": 1021, "K": 2560, "H": 6912, "E": 4, "empty": 0, "dtype": "bf16"},
        {"name": "ffn 16384 rows", "op": "ffn", "rows": 16384, "K": 2560, "H": 6912, "E": 4, "empty": 0, "dtype": "bf16"},
    ]


def draw(rng):
    def spread(lo, hi, step=1):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))

    op = rng.choice(("cast", "linear", "linear", "grouped", "grouped", "ffn", "ffn"))
    case = {"op": op, "dtype": rng.choice(("bf16", "fp16"))}
    if op == "cast":
        return dict(case, rows=spread(1, 32768), K=spread(128, 6912, 16))
    if op == "linear":
        return dict(case, rows=spread(1, 16384), K=spread(512, 6912, 16), N=spread(512, 6912, 16), bias=rng.random() < 0.5)
    E = rng.choice((2, 3, 4, 6, 8, 16))
    case.update(rows=spread(2, 16384), K=spread(512, 4096, 16), E=E, empty=rng.choice((0, 0, 1, E // 2)))
    if op == "grouped":
        return dict(case, N=spread(512, 8192, 16))
    return dict(case, H=spread(512, 4096, 16))


def _weight(gen, E, n, k):
    """E weights [n, k] as e4m3fn values and one scale for each 128 x 128 block of them."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    spread = torch.rand((E, nb, 1, kb, 1), generator=gen, device="cuda") + 0.5
    w = torch.randn((E, nb, BLOCK, kb, BLOCK), generator=gen, device="cuda") * (spread / math.sqrt(k))
    s = w.abs().amax((2, 4), keepdim=True) / 448
    q = (w / s).reshape(E, nb * BLOCK, kb * BLOCK)[:, :n, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), s.reshape(E, nb, kb).contiguous()


def _offsets(gen, rows, E, empty):
    """Bounds of the experts' row segments, of uneven sizes, `empty` of them without rows; and the longest one."""
    share = torch.rand(E, generator=gen, dtype=torch.float64) + 0.25
    share[torch.randperm(E, generator=gen)[:empty]] = 0
    ends = (share.cumsum(0) / share.sum() * rows).round().to(torch.int64)
    ends[-1] = rows
    bounds = torch.cat([torch.zeros(1, dtype=torch.int64), ends])
    return bounds.to(torch.int32).cuda(), int((bounds[1:] - bounds[:-1]).max())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, K, dtype = case["rows"], case["K"], DTYPES[case["dtype"]]
    # activations with channels of very different size, as those behind a modulated norm have
    channel = torch.exp(0.7 * torch.randn(K, generator=gen, device="cuda"))
    x = (torch.randn((rows, K), generator=gen, device="cuda") * channel).to(dtype)
    s = {"case": dict(case), "x": x}
    if case["op"] == "cast":
        return s
    if case["op"] == "linear":
        w, sw = _weight(gen, 1, case["N"], K)
        s["bias"] = torch.randn(case["N"], generator=gen, device="cuda").to(dtype) if case["bias"] else None
        s["w"], s["sw"] = w[0], sw[0]
        return s
    E = case["E"]
    s["offsets"], s["longest"] = _offsets(torch.Generator().manual_seed(seed), rows, E, case["empty"])
    if case["op"] == "grouped":
        s["w"], s["sw"] = _weight(gen, E, case["N"], K)
        s["experts"] = [(s["w"][e], s["sw"][e], None) for e in range(E)]
        return s
    for name, n, k in (("1", case["H"], K), ("3", case["H"], K), ("2", K, case["H"])):
        s["w" + name], s["sw" + name] = _weight(gen, E, n, k)
    s["gate_up"] = [(s["w1"][e], s["sw1"][e], s["w3"][e], s["sw3"][e]) for e in range(E)]
    s["down"] = [(s["w2"][e], s["sw2"][e], None) for e in range(E)]
    return s


def _cast(x):
    """q as e4m3fn and s for the rows of x, in 32 bits."""
    rows, K = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).reshape(rows, -1, BLOCK)
    top = blocks.abs().amax(-1, keepdim=True).clamp_min(FLOOR)
    most = torch.full_like(top, 448.0)   # tensors on both sides: torch multiplies by the reciprocal of a number
    q = (blocks * (most / top)).to(torch.float8_e4m3fn).reshape(rows, -1)[:, :K]
    return q.contiguous(), (top / most)[..., 0]


def _rows(q, s):
    return q.float() * s.repeat_interleave(BLOCK, -1)[:, :q.shape[1]]


def _matrix(w, sw):
    """The values of weights [..., n, k] from their codes and scales."""
    n, k = w.shape[-2:]
    return w.float() * sw.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _groups(s):
    """Row numbers [E, longest] of the experts' segments (past a segment's end: the last row), and each row's place in that."""
    o, rows = s["offsets"].long(), s["case"]["rows"]
    at = torch.arange(s["longest"], device=o.device)
    row = torch.arange(rows, device=o.device)
    e = torch.searchsorted(o[1:].contiguous(), row, right=True)
    return (o[:-1, None] + at).clamp_max(rows - 1), e * s["longest"] + row - o[e]


def _grouped(x, idx, place, w):
    return torch.matmul(x[idx], w.transpose(1, 2)).flatten(0, 1)[place]


def _plain(s):
    case, x = s["case"], s["x"]
    q, sx = _cast(x)
    if case["op"] == "cast":
        return q, sx
    if case["op"] == "linear":
        y = torch.matmul(_rows(q, sx), _matrix(s["w"], s["sw"]).t())
        return (y if s["bias"] is None else y + s["bias"].float()).to(x.dtype)
    idx, place = _groups(s)
    if case["op"] == "grouped":
        return _grouped(_rows(q, sx), idx, place, _matrix(s["w"], s["sw"])).to(x.dtype)
    xr = _rows(q, sx)
    g, u = (_grouped(xr, idx, place, _matrix(s["w" + n], s["sw" + n])) for n in "13")
    h = _rows(*_cast(g / (1 + torch.exp(-g)) * u))
    return _grouped(h, idx, place, _matrix(s["w2"], s["sw2"])).to(x.dtype)


def run(state):
    if not own:
        return _plain(state)
    from comfyui_amd import functional as HF
    op, x = state["case"]["op"], state["x"]
    if op == "cast":
        return HF.quant_block_fp8(x)
    if op == "linear":
        return HF.linear_block_fp8(x, state["w"], state["sw"], bias=state["bias"])
    if op == "grouped":
        return HF.grouped_linear_block_fp8(x, state["offsets"], state["experts"])
    h, sh = HF.grouped_swiglu_block_fp8(x, state["offsets"], state["gate_up"])
    return HF.grouped_linear_block_fp8(h, state["offsets"], state["down"], scale_a=sh, out_dtype=x.dtype)


def work(case):
    op, rows, K = case["op"], case["rows"], case["K"]
    blocks = lambda n: -(-n // BLOCK)  # noqa: E731
    if op == "cast":
        return {"bytes": rows * (3 * K + 4 * blocks(K)), "flops": 0}
    # experts that can have rows: each of them is counted as read
    E = 1 if op == "linear" else min(case["E"] - case["empty"], rows)
    if op == "ffn":
        H = case["H"]
        return {"bytes": E * 3 * (H * K + 4 * blocks(H) * blocks(K)) + 4 * rows * K, "flops": 6 * rows * K * H}
    N = case["N"]
    return {"bytes": E * (N * K + 4 * blocks(N) * blocks(K)) + 2 * rows * (K + N) + (2 * N if case.get("bias") else 0),
            "flops": 2 * rows * K * N}


def exact(case, seed):
    """From the definitions, in 64 bits, one expert and one block of columns at a time. The scales are 32-bit numbers by
    definition (quotients of two), and so is the product that a cast of 16-bit values rounds."""
    s = prepare(case, seed)

    def cast(v, narrow):
        q, t = torch.empty_like(v), torch.empty((v.shape[0], -(-v.shape[1] // BLOCK)), dtype=torch.float64, device=v.device)
        for b in range(t.shape[1]):
            part = v[:, b * BLOCK:(b + 1) * BLOCK]
            top = torch.maximum(part.abs().max(1).values, torch.tensor(FLOOR, dtype=torch.float64, device=v.device))
            r = (448.0 / top).float().double() if narrow else 448.0 / top
            z = part * r[:, None]
            q[:, b * BLOCK:(b + 1) * BLOCK] = (z.float() if narrow else z).to(torch.float8_e4m3fn).double()
            t[:, b] = (top / 448.0).float().double() if narrow else top / 448.0
        return q, t

    def product(q, t, w, sw):
        y = torch.zeros((q.shape[0], w.shape[0]), dtype=torch.float64, device=q.device)
        per_row = sw.double().repeat_interleave(BLOCK, 0)[:w.shape[0]]
        for b in range(t.shape[1]):
            cols = slice(b * BLOCK, (b + 1) * BLOCK)
            y += (q[:, cols] * t[:, b:b + 1]) @ (w[:, cols].double() * per_row[:, b:b + 1]).t()
        return y

    q, t = cast(s["x"].double(), True)
    if case["op"] == "cast":
        return q, t
    if case["op"] == "linear":
        y = product(q, t, s["w"], s["sw"])
        return y if s["bias"] is None else y + s["bias"].double()
    bounds = s["offsets"].tolist()
    width = case["N"] if case["op"] == "grouped" else case["K"]
    y = torch.zeros((case["rows"], width), dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        lo, hi = bounds[e], bounds[e + 1]
        if hi <= lo:
            continue
        if case["op"] == "grouped":
            y[lo:hi] = product(q[lo:hi], t[lo:hi], s["w"][e], s["sw"][e])
            continue
        g, u = (product(q[lo:hi], t[lo:hi], s["w" + n][e], s["sw" + n][e]) for n in "13")
        h, th = cast(g * torch.sigmoid(g) * u, False)
        y[lo:hi] = product(h, th, s["w2"][e], s["sw2"][e])
    return y
