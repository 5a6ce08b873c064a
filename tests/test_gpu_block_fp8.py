"""e4m3fn Linears with a scale for each block of 128 against their definition in 64 bits.

Tolerances. A 16-bit output is off by half a step (2^-8 of the value in bf16, 2^-11 in fp16) and by what the sums before it are.
The fp8 matrix instruction adds eight neighbouring products at a time, each cut off (towards zero) at 2^-13 of the largest one's
power of two: 256 * 256 + 2^3 in a group of eight comes out exactly, + 2^2 (and 7 times 2^2) as 256 * 256, and in another group + 2^-7
still counts. So a group is off by less than 7 * 2^-13 of its largest product. The groups' sums, at most 16 in an instruction and then one
a block, add in fp32, cut or rounded: 2^-23 of the partial sum each, with 16 + 2 * 64 of them 2^-15.8 of the sum of magnitudes.
`product64` returns these two as `err` beside the 64-bit product.
A cast output h is compared with the unrounded 64-bit value: half an e4m3fn step is 2^-4 of the value, or 2^-10 of the scale below
the normal range; the error of the value itself and that of the scale come on top."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128
FLOOR = 2.0 ** -96
F8 = torch.float8_e4m3fn
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def nb(n):
    return -(-n // BLOCK)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weight(g, n, k):
    """A random e4m3fn weight and block scales of very different size."""
    w = (torch.randn((n, k), generator=g, device="cuda") * 60).clamp(-440, 440).to(F8)
    s = torch.exp(torch.randn((nb(n), nb(k)), generator=g, device="cuda")) * (0.02 / k ** 0.5)
    return w, s


def tokens(g, rows, k, dtype=torch.bfloat16):
    channel = torch.exp(torch.randn(k, generator=g, device="cuda"))
    return (torch.randn((rows, k), generator=g, device="cuda") * channel).to(dtype)


def cast_cpu(x):
    """The definition on the CPU, in fp32 throughout (tensor by tensor: torch multiplies by the reciprocal of a number)."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x.cpu().float(), (0, -k % BLOCK)).reshape(rows, nb(k), BLOCK)
    top = b.abs().amax(-1, keepdim=True).clamp_min(FLOOR)
    most = torch.full_like(top, 448.0)
    return (b * (most / top)).to(F8).reshape(rows, -1)[:, :k], (top / most)[..., 0]


def rows64(q, s):
    return q.double() * s.double().repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def matrix64(w, s):
    return w.double() * s.double().repeat_interleave(BLOCK, 0)[:w.shape[0]].repeat_interleave(BLOCK, 1)[:, :w.shape[1]]


def product64(q, s, w, sw, bias=None, exact=False):
    """The product in 64 bits and how far the device's sums may be from it (exact: with products that are not cut)."""
    a, m = rows64(q, s), matrix64(w, sw)
    y = a @ m.t()
    err = (a.abs() @ m.abs().t()) * 2.0 ** -15.8
    if bias is not None:
        y, err = y + bias.double(), err + bias.double().abs() * 2.0 ** -23
    if exact:
        return y, err
    a8, m8 = a.abs().float(), m.abs().float()
    largest = torch.zeros_like(y, dtype=torch.float32)
    for k in range(0, a.shape[1], 8):
        top = a8[:, None, k] * m8[None, :, k]
        for j in range(k + 1, k + 8):
            top = torch.maximum(top, a8[:, None, j] * m8[None, :, j])
        largest += top
    return y, err + largest.double() * (7 * 2.0 ** -13 * (1 + 2.0 ** -10))


def close(y, want, err):
    limit = STEP[y.dtype] * (want.abs() + err) + err
    over = ((y.double() - want).abs() - limit * (1 + 2.0 ** -7)).max()
    assert over <= 0, f"off by {over.item():.3g} more than allowed"


def silu64(v):
    return v * torch.sigmoid(v)


def close_cast(h, sh, q, s, w1, s1, w3, s3, exact=False):
    """h, sh against the unrounded 64-bit silu(g) * u of the same cast rows."""
    (gt, gm), (u, um) = product64(q, s, w1, s1, exact=exact), product64(q, s, w3, s3, exact=exact)
    want = silu64(gt) * u
    # |silu'| <= 1.1; the fp32 exp, quotient and product add a few 2^-23 of the value, and |g| 2^-22 of it the exponent's rounding
    err = 1.1 * gm * (u.abs() + um) + silu64(gt).abs() * um + (2.0 ** -20 + gt.abs() * 2.0 ** -22) * want.abs()
    rows, H = h.shape
    pad = lambda t: torch.nn.functional.pad(t, (0, -H % BLOCK)).reshape(rows, nb(H), BLOCK)  # noqa: E731
    top = pad(want.abs()).amax(-1).clamp_min(FLOOR)
    assert ((sh.double() - top / 448).abs() <= (pad(err).amax(-1) + 2.0 ** -22 * top) / 448).all(), "scales"
    got = h.double() * sh.double().repeat_interleave(BLOCK, 1)[:, :H]
    per = sh.double().repeat_interleave(BLOCK, 1)[:, :H]
    limit = 2.0 ** -4 * want.abs() + 2.0 ** -10 * per + err * (1 + 2.0 ** -4)
    over = ((got - want).abs() - limit * (1 + 2.0 ** -7)).max()
    assert over <= 0, f"off by {over.item():.3g} more than allowed"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 16), (1, 128), (3, 144), (17, 2560), (65, 1040), (257, 6912), (1000, 336)])
def test_cast(rows, K, dtype):
    from comfyui_amd import functional as HF
    x = tokens(gen(rows + K), rows, K, dtype)
    x[rows // 2] = 0
    x[0, K // 2] *= 100
    q, s = HF.quant_block_fp8(x)
    q_ref, s_ref = cast_cpu(x)
    assert q.shape == x.shape and s.shape == (rows, nb(K)) and s.stride(0) == 1
    assert torch.equal(s.cpu(), s_ref)
    assert torch.equal(q.cpu().view(torch.uint8), q_ref.contiguous().view(torch.uint8))


def test_cast_of_tiny_huge_and_non_finite_blocks():
    from comfyui_amd import functional as HF
    x = torch.zeros((6, 256), dtype=torch.bfloat16, device="cuda")
    x[0, :] = 1e-38                      # below the floor of the scale
    x[1, 5] = 3e38
    x[2, 7] = float("inf")
    x[3, 200] = float("nan")
    x[4, 3] = float("-inf")
    x[5, 130:140] = -2.0
    q, s = HF.quant_block_fp8(x)
    q_ref, s_ref = cast_cpu(x)
    assert torch.equal(s.cpu()[[0, 1, 5]], s_ref[[0, 1, 5]]) and torch.isfinite(s[[0, 1, 5]]).all()
    same = q.cpu().float() == q_ref.float()
    assert same[[0, 1, 5]].all()
    for r, b in ((2, 0), (3, 1), (4, 0)):
        other = 1 - b
        assert not torch.isfinite(s[r, b]) and s[r, other] == s_ref[r, other]
        block = q.float()[r, b * 128:b * 128 + 128].cpu()
        assert torch.isnan(block[[7, 72, 3][[2, 3, 4].index(r)]])
    w, sw = weight(gen(1), 32, 256)
    y = HF.linear_block_fp8(x, w, sw)
    assert torch.isnan(y[[2, 3, 4]]).all() and torch.isfinite(y[[0, 5]]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("rows,K,N", [(1, 16, 16), (1, 2560, 6912), (2, 640, 240), (5, 128, 128), (16, 1040, 272), (17, 2560, 512),
                                      (31, 384, 784), (33, 144, 1040), (48, 6912, 2560), (64, 512, 256), (65, 2064, 528),
                                      (128, 1280, 1296), (129, 256, 400), (200, 656, 2064), (256, 2560, 256), (257, 784, 640),
                                      (300, 3600, 1808), (1021, 2048, 1024), (2050, 512, 2560)])
def test_linear(rows, K, N, bias, dtype):
    from comfyui_amd import functional as HF
    g = gen(rows * 7 + K + N)
    x = tokens(g, rows, K, dtype)
    w, sw = weight(g, N, K)
    b = torch.randn(N, generator=g, device="cuda").to(dtype) if bias else None
    y = HF.linear_block_fp8(x, w, sw, bias=b)
    assert y.dtype == dtype and y.shape == (rows, N)
    q, s = HF.quant_block_fp8(x)
    close(y, *product64(q, s, w, sw, b))
    # cast rows give the same: with the scales as they come and laid out row by row
    for scales in (s, s.contiguous()):
        y2 = HF.linear_block_fp8(q, w, sw, bias=b, scale_x=scales, out_dtype=dtype)
        close(y2, *product64(q, s, w, sw, b))


def test_linear_reads_nothing_but_its_own_rows():
    """Rows, weights and scales behind the last ones hold NaN: none of it may reach an output (short blocks and tiles)."""
    from comfyui_amd import functional as HF
    for rows, K, N in ((3, 144, 144), (70, 400, 272), (300, 656, 1040)):
        g = gen(rows)
        x = tokens(g, rows, K)
        w, sw = weight(g, N, K)
        q, s = HF.quant_block_fp8(x)
        want = product64(q, s, w, sw)
        nan8 = torch.full(((rows + 5) * K + 4096,), 0x7f, dtype=torch.uint8, device="cuda").view(F8)
        qq = nan8[:rows * K].view(rows, K)
        qq.copy_(q)
        nw = torch.full((N * K + 65536,), 0x7f, dtype=torch.uint8, device="cuda").view(F8)
        ww = nw[:N * K].view(N, K)
        ww.copy_(w)
        ns = torch.full((sw.numel() + 512,), float("nan"), device="cuda")
        sww = ns[:sw.numel()].view(sw.shape)
        sww.copy_(sw)
        na = torch.full((s.numel() + 512,), float("nan"), device="cuda")
        ss = na[:s.numel()].view(nb(K), rows).t()
        ss.copy_(s)
        close(HF.linear_block_fp8(qq, ww, sww, scale_x=ss), *want)


def segments(sizes):
    return torch.tensor([0] + list(torch.tensor(sizes).cumsum(0)), dtype=torch.int32, device="cuda")


GROUPS = [([1], 128, 256), ([0, 2, 0, 0], 2560, 512), ([1, 1, 1, 1], 640, 272), ([5, 0, 16, 17, 1, 0, 33, 2], 400, 784),
          ([0, 0, 0], 128, 128), ([64, 64, 0, 128], 1040, 1040), ([130, 7, 0, 255, 256, 257, 1, 94], 512, 528),
          ([1000, 3, 500], 1296, 640), ([7] * 32, 272, 144)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,K,N", GROUPS)
def test_grouped_linear(sizes, K, N, dtype):
    from comfyui_amd import functional as HF
    g = gen(sum(sizes) + K)
    rows = sum(sizes)
    x = tokens(g, rows, K, dtype)
    experts = [(*weight(g, N, K), torch.randn(N, generator=g, device="cuda").to(dtype) if e % 2 else None) for e in range(len(sizes))]
    off = segments(sizes)
    y = HF.grouped_linear_block_fp8(x, off, experts)
    assert y.shape == (rows, N) and y.dtype == dtype
    q, s = HF.quant_block_fp8(x)
    b = off.tolist()
    for e, (w, sw, bias) in enumerate(experts):
        lo, hi = b[e], b[e + 1]
        if hi > lo:
            close(y[lo:hi], *product64(q[lo:hi], s[lo:hi], w, sw, bias))


@pytest.mark.parametrize("sizes,K,H", GROUPS)
def test_grouped_swiglu(sizes, K, H):
    from comfyui_amd import functional as HF
    g = gen(sum(sizes) + H)
    rows = sum(sizes)
    x = tokens(g, rows, K)
    experts = [(*weight(g, H, K), *weight(g, H, K)) for _ in sizes]
    off = segments(sizes)
    h, sh = HF.grouped_swiglu_block_fp8(x, off, experts)
    assert h.shape == (rows, H) and h.dtype == F8 and sh.shape == (rows, nb(H))
    q, s = HF.quant_block_fp8(x)
    b = off.tolist()
    for e, ws in enumerate(experts):
        lo, hi = b[e], b[e + 1]
        if hi > lo:
            close_cast(h[lo:hi], sh[lo:hi], q[lo:hi], s[lo:hi], *ws)


@pytest.mark.parametrize("T,K,H,Hs,E", [(1, 512, 256, 128, 4), (9, 656, 272, 400, 3), (150, 512, 768, 384, 4), (700, 512, 640, 256, 8)])
def test_feed_forward_of_a_layer(T, K, H, Hs, E):
    """Both halves as a layer runs them: routed rows read through the permutation, the shared expert in the same launches."""
    from comfyui_amd import functional as HF
    g = gen(T)
    x = tokens(g, T, K)
    idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:2] for t in range(T)]).to(torch.int32).cuda()
    counts, off, perm, inv = HF.dispatch(idx, E)
    up = [(*weight(g, H, K), *weight(g, H, K)) for _ in range(E)]
    down = [(*weight(g, K, H), None) for _ in range(E)]
    up_s, down_s = (*weight(g, Hs, K), *weight(g, Hs, K)), (*weight(g, K, Hs), None)
    q, s = HF.quant_block_fp8(x)
    h, sh, hs, shs = HF.grouped_swiglu_block_fp8(q, off, up, scale_a=s, perm=perm, shared=up_s)
    y, ys = HF.grouped_linear_block_fp8(h, off, down, scale_a=sh, shared=down_s, a_static=hs, scale_static=shs)
    rows = perm.long() // 2
    b = off.tolist()
    for e in range(E):
        lo, hi = b[e], b[e + 1]
        if hi > lo:
            close_cast(h[lo:hi], sh[lo:hi], q[rows[lo:hi]], s[rows[lo:hi]], *up[e])
            close(y[lo:hi], *product64(h[lo:hi], sh[lo:hi], *down[e]))
    close_cast(hs, shs, q, s, *up_s)
    close(ys, *product64(hs, shs, *down_s))
    # the first product through the permutation, without the activation
    first = [(w, sw, None) for w, sw, _, _ in up]
    z = HF.grouped_linear_block_fp8(x, off, first, perm=perm)
    for e in range(E):
        lo, hi = b[e], b[e + 1]
        if hi > lo:
            close(z[lo:hi], *product64(q[rows[lo:hi]], s[rows[lo:hi]], *first[e]))


def test_rows_in_no_segment_are_left_alone():
    """Segments that start late, end early or point past the rows: what lies in none is not written, nothing else is read."""
    from comfyui_amd import _lib
    from comfyui_amd import functional as HF
    for rows in (40, 300):
        g = gen(rows)
        K, N, E = 272, 400, 2
        x = tokens(g, rows, K)
        q, s = HF.quant_block_fp8(x)
        ws = [weight(g, N, K) for _ in range(E)]
        for bounds in ([3, 9, rows - 5], [0, 0, rows + 1000], [-7, 4, 4], [rows, rows, rows]):
            off = torch.tensor(bounds, dtype=torch.int32, device="cuda")
            out = torch.full((rows, N), 7.0, dtype=torch.bfloat16, device="cuda")
            args = _lib.BlockArgs()
            args.a_dtype, args.out_dtype = _lib.W_E4M3FN, _lib.W_BF16
            args.E, args.rows, args.K, args.N = E, rows, K, N
            args.offsets = off.data_ptr()
            args.experts = (_lib.BlockWeights * E)(*(_lib.BlockWeights(w.data_ptr(), sw.data_ptr(), None, None, None) for w, sw in ws))
            args.routed = _lib.BlockRows(q.data_ptr(), s.data_ptr(), rows, out.data_ptr(), None, 0)
            _lib.check(_lib.lib.hdmoe_block_linear(ctypes.byref(args), torch.cuda.current_stream().cuda_stream))
            b = [min(max(v, 0), rows) for v in bounds]
            for e in range(E):
                if b[e + 1] > b[e]:
                    close(out[b[e]:b[e + 1]], *product64(q[b[e]:b[e + 1]], s[b[e]:b[e + 1]], *ws[e]))
            assert (out[:b[0]] == 7).all() and (out[b[-1]:] == 7).all()


def test_a_bad_index_of_the_permutation_reads_as_zeros():
    from comfyui_amd import functional as HF
    g = gen(5)
    T, K, N = 20, 256, 256
    x = tokens(g, T, K)
    w, sw = weight(g, N, K)
    perm = torch.arange(2 * T, dtype=torch.int32, device="cuda")
    perm[3], perm[4], perm[5] = 2 * T, -1, 2 ** 31 - 1
    y = HF.grouped_linear_block_fp8(x, segments([2 * T]), [(w, sw, None)], perm=perm)
    assert (y[3:6] == 0).all()
    q, s = HF.quant_block_fp8(x)
    keep = [r for r in range(2 * T) if r not in (3, 4, 5)]
    at = torch.tensor([r // 2 for r in keep], device="cuda")
    close(y[torch.tensor(keep, device="cuda")], *product64(q[at], s[at], w, sw))


def test_captured_into_a_graph():
    """Both halves captured together and replayed on new inputs, with eager work between the replays."""
    from comfyui_amd import functional as HF
    for rows in (6, 40, 700):
        g = gen(rows)
        K, H, E = 512, 384, 3
        up = [(*weight(g, H, K), *weight(g, H, K)) for _ in range(E)]
        down = [(*weight(g, K, H), None) for _ in range(E)]
        w, sw = weight(g, 272, K)
        off = segments([rows // 2, 0, rows - rows // 2])
        x = tokens(g, rows, K)

        def run(t):
            h, sh = HF.grouped_swiglu_block_fp8(t, off, up)
            y = HF.grouped_linear_block_fp8(h, off, down, scale_a=sh)
            return y, HF.linear_block_fp8(y, w, sw)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        static = x.clone()
        with torch.cuda.graph(graph):
            outs = run(static)
        for k in range(4):
            fresh = tokens(gen(100 + k), rows, K)
            static.copy_(fresh)
            graph.replay()
            want = run(fresh)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), f"replay {k}"


def test_on_another_stream_and_twice_at_once():
    """Calls on two streams share nothing: the same bytes as one after the other."""
    from comfyui_amd import functional as HF
    g = gen(9)
    for rows in (4, 300):
        xs = [tokens(g, rows, 1296) for _ in range(2)]
        ws = [weight(g, 784, 1296) for _ in range(2)]
        want = [HF.linear_block_fp8(x, *w) for x, w in zip(xs, ws)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = [[], []]
        for _ in range(10):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(HF.linear_block_fp8(xs[i], *ws[i]))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_no_rows():
    from comfyui_amd import functional as HF
    g = gen(2)
    w, sw = weight(g, 256, 128)
    x = torch.empty((0, 128), dtype=torch.bfloat16, device="cuda")
    q, s = HF.quant_block_fp8(x)
    assert q.shape == (0, 128) and s.shape == (0, 1)
    assert HF.linear_block_fp8(x, w, sw).shape == (0, 256)
    assert HF.grouped_linear_block_fp8(x, segments([0, 0]), [(w, sw, None)] * 2).shape == (0, 256)
    h, sh = HF.grouped_swiglu_block_fp8(x, segments([0]), [(w, sw, w, sw)])
    assert h.shape == (0, 256) and sh.shape == (0, 2)


def uneven(rows, n):
    """Sizes of n segments, the first about half of the rows, the second empty where there are more than three."""
    if n == 0:
        return []
    left, sizes = rows, []
    for i in range(n):
        take = left if i == n - 1 else 0 if i == 1 and n > 3 else -(-left // 2)
        sizes.append(take)
        left -= take
    return sizes


# Sizes at which each way to run a contraction is taken: few rows with 1, 2 and 4 tiles of 16 rows by 1, 2 and 4 strips of weights, with and
# without the cast inside; 128-row tiles with 2 and 4 steps on their way; 256-row ones of up to 2, 3 and 4 parts
EVERY = [(5, 0, 608, 64), (30, 3, 320, 64), (12, 0, 704, 64), (42, 3, 208, 64), (558, 0, 176, 160), (1285, 3, 240, 80), (292, 0, 144, 224),
         (495, 3, 144, 144), (77, 0, 144, 3136), (544, 3, 304, 448), (1494, 0, 176, 96), (3774, 3, 144, 64), (1584, 0, 400, 80), (852, 3, 352, 144),
         (1621, 0, 144, 112), (2544, 6, 160, 64), (1695, 0, 144, 192), (1717, 6, 144, 224), (33, 0, 144, 3056), (119, 3, 160, 1104),
         (916, 0, 240, 544), (165, 3, 160, 1392), (1017, 0, 144, 528), (2134, 3, 160, 288), (3807, 3, 2128, 4080), (3440, 0, 880, 3552),
         (3356, 3, 1040, 3312), (3980, 0, 832, 3888), (3888, 3, 736, 3808), (2908, 0, 208, 336), (3413, 3, 192, 320), (3666, 0, 1936, 304),
         (2959, 3, 2000, 336), (100, 0, 6912, 272), (3, 0, 5360, 400), (20, 4, 16400, 96), (1, 0, 16400, 144)]
EVERY_GATE_UP = [(5, 0, 592, 64), (36, 3, 272, 80), (5, 0, 480, 64), (62, 3, 192, 80), (202, 0, 288, 608), (193, 3, 416, 576), (290, 0, 144, 224),
                 (1224, 3, 400, 64), (854, 0, 272, 96), (230, 3, 352, 272), (1214, 0, 272, 144), (843, 3, 288, 176), (46, 0, 288, 2256),
                 (1608, 3, 304, 144), (1143, 0, 304, 240), (1760, 6, 288, 144), (3128, 0, 144, 688), (3498, 3, 144, 592), (3117, 0, 160, 1312),
                 (1969, 3, 144, 1984), (1997, 0, 160, 2976), (3374, 3, 144, 1680), (10, 0, 176, 80), (69, 3, 224, 64), (3, 0, 5360, 272), (20, 4, 8208, 96)]


@pytest.mark.parametrize("rows,E,K,N", EVERY)
def test_linear_every_way(rows, E, K, N):
    from comfyui_amd import functional as HF
    g = gen(rows + K + N)
    x = tokens(g, rows, K)
    q, s = HF.quant_block_fp8(x)
    sizes = uneven(rows, E) or [rows]
    experts = [(*weight(g, N, K), None) for _ in sizes]
    off = segments(sizes)
    b = off.tolist()
    for a, scale in ((x, None), (q, s)):
        y = HF.grouped_linear_block_fp8(a, off, experts, scale_a=scale) if E else HF.linear_block_fp8(a, *experts[0][:2], scale_x=scale)
        for e, (w, sw, _) in enumerate(experts):
            lo, hi = b[e], b[e + 1]
            if hi > lo:
                close(y[lo:hi], *product64(q[lo:hi], s[lo:hi], w, sw, None))


@pytest.mark.parametrize("rows,E,K,N", EVERY_GATE_UP)
def test_swiglu_every_way(rows, E, K, N):
    from comfyui_amd import functional as HF
    g = gen(rows + K + N)
    x = tokens(g, rows, K)
    q, s = HF.quant_block_fp8(x)
    sizes = uneven(rows, E) or [rows]
    experts = [(*weight(g, N, K), *weight(g, N, K)) for _ in sizes]
    off = segments(sizes)
    b = off.tolist()
    for a, scale in ((x, None), (q, s)):
        h, sh = HF.grouped_swiglu_block_fp8(a, off, experts, scale_a=scale) if E else HF.swiglu_block_fp8(a, *experts[0], scale_x=scale)
        for e, ws in enumerate(experts):
            lo, hi = b[e], b[e + 1]
            if hi > lo:
                close_cast(h[lo:hi], sh[lo:hi], q[lo:hi], s[lo:hi], *ws)


@pytest.mark.parametrize("sizes,K,N", [([700, 130, 0, 300, 65, 500], 1552, 7696), ([900, 64, 330], 1040, 6800), ([257] * 5, 1040, 7952),
                                       ([1500, 1100, 700], 656, 5264), ([200, 520, 90, 700], 656, 5264), ([1300, 40, 40], 528, 4624), ([480, 0, 700, 350, 420, 600, 250, 201], 2064, 8176)])
def test_more_tiles_than_cus(sizes, K, N):
    """Tiles of different heights, up to two for every CU and a few more."""
    test_grouped_linear(sizes, K, N, torch.bfloat16)
    test_grouped_swiglu(sizes, K, N // 2 // 16 * 16)


@pytest.mark.parametrize("rows,E,K,N", EVERY_GATE_UP)
def test_swiglu_of_fp16_has_exact_products(rows, E, K, N):
    """Products and sums of fp16 activations' gate/up are fp32: within 2^-15.8 of the sum of magnitudes, without what the e4m3fn instruction cuts."""
    from comfyui_amd import functional as HF
    g = gen(rows + K + N)
    x = tokens(g, rows, K, torch.float16)
    q, s = HF.quant_block_fp8(x)
    sizes = uneven(rows, E) or [rows]
    experts = [(*weight(g, N, K), *weight(g, N, K)) for _ in sizes]
    off = segments(sizes)
    b = off.tolist()
    h, sh = HF.grouped_swiglu_block_fp8(x, off, experts) if E else HF.swiglu_block_fp8(x, *experts[0])
    for e, ws in enumerate(experts):
        lo, hi = b[e], b[e + 1]
        if hi > lo:
            close_cast(h[lo:hi], sh[lo:hi], q[lo:hi], s[lo:hi], *ws, exact=True)


@pytest.mark.parametrize("rows,E,K,N", [(1, 0, 2560, 6912), (2, 4, 2560, 1040), (5, 0, 592, 64), (36, 3, 272, 80), (48, 3, 656, 400), (16, 0, 6912, 272)])
def test_swiglu_of_few_rows_has_exact_products(rows, E, K, N):
    """So it is in bf16 where the few-row kernels run."""
    from comfyui_amd import functional as HF
    g = gen(rows + K + N)
    x = tokens(g, rows, K)
    q, s = HF.quant_block_fp8(x)
    sizes = uneven(rows, E) or [rows]
    experts = [(*weight(g, N, K), *weight(g, N, K)) for _ in sizes]
    off = segments(sizes)
    b = off.tolist()
    for a, scale in ((x, None), (q, s)):
        h, sh = HF.grouped_swiglu_block_fp8(a, off, experts, scale_a=scale) if E else HF.swiglu_block_fp8(a, *experts[0], scale_x=scale)
        for e, ws in enumerate(experts):
            lo, hi = b[e], b[e + 1]
            if hi > lo:
                close_cast(h[lo:hi], sh[lo:hi], q[lo:hi], s[lo:hi], *ws, exact=True)
