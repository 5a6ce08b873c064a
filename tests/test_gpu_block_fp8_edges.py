"""Calls of the block-scaled contractions at the ends of what they allow: many experts with a shared one, bounds outside the rows, the same row
twice, outputs of more than 2^31 elements, two captured graphs replayed in turn, weights that are views."""
import pytest
import torch

from tests.test_gpu_block_fp8 import F8, close, close_cast, gen, product64, segments, tokens, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,K,H,Hs", [(40, 272, 144, 400), (900, 272, 656, 1040), (3000, 528, 784, 656)])
def test_32_experts_and_a_shared_one(T, K, H, Hs):
    from comfyui_amd import functional as HF
    g = gen(T)
    E = 32
    x = tokens(g, T, K)
    q, s = HF.quant_block_fp8(x)
    perm = torch.randperm(2 * T, generator=torch.Generator().manual_seed(T)).to(torch.int32).cuda()
    ends = torch.sort(torch.randint(0, 2 * T + 1, (E - 1,), generator=torch.Generator().manual_seed(T))).values.tolist()
    b = [0] + ends + [2 * T]
    off = torch.tensor(b, dtype=torch.int32, device="cuda")
    up = [(*weight(g, H, K), *weight(g, H, K)) for _ in range(E)]
    up_s = (*weight(g, Hs, K), *weight(g, Hs, K))
    down = [(*weight(g, K, H), None) for _ in range(E)]
    down_s = (*weight(g, K, Hs), None)
    rows = perm.long() // 2
    for a, scale in ((x, None), (q, s)):
        h, sh, hs, shs = HF.grouped_swiglu_block_fp8(a, off, up, scale_a=scale, perm=perm, shared=up_s)
        y, ys = HF.grouped_linear_block_fp8(h, off, down, scale_a=sh, shared=down_s, a_static=hs, scale_static=shs)
        for e in range(E):
            lo, hi = b[e], b[e + 1]
            if hi > lo:
                close_cast(h[lo:hi], sh[lo:hi], q[rows[lo:hi]], s[rows[lo:hi]], *up[e])
                close(y[lo:hi], *product64(h[lo:hi], sh[lo:hi], *down[e]))
        close_cast(hs, shs, q, s, *up_s)
        close(ys, *product64(hs, shs, *down_s))


@pytest.mark.parametrize("rows", [7, 90, 700])
def test_bounds_outside_the_rows_are_cut_off(rows):
    from comfyui_amd import functional as HF
    g = gen(rows)
    x = tokens(g, rows, 400)
    q, s = HF.quant_block_fp8(x)
    experts = [(*weight(g, 272, 400), None) for _ in range(3)]
    up = [(*weight(g, 272, 400), *weight(g, 272, 400)) for _ in range(3)]
    mid = rows // 2
    off = torch.tensor([-7, mid, rows + 5, 2 ** 30], dtype=torch.int32, device="cuda")
    y = HF.grouped_linear_block_fp8(x, off, experts)
    h, sh = HF.grouped_swiglu_block_fp8(x, off, up)
    for e, (lo, hi) in enumerate(((0, mid), (mid, rows))):
        close(y[lo:hi], *product64(q[lo:hi], s[lo:hi], *experts[e]))
        close_cast(h[lo:hi], sh[lo:hi], q[lo:hi], s[lo:hi], *up[e])


@pytest.mark.parametrize("T", [1, 30, 400])
def test_the_same_token_many_times(T):
    from comfyui_amd import functional as HF
    g = gen(T)
    x = tokens(g, T, 528)
    w = weight(g, 272, 528)
    perm = torch.full((2 * T,), 2 * (T - 1) + 1, dtype=torch.int32, device="cuda")
    y = HF.grouped_linear_block_fp8(x, segments([2 * T]), [(*w, None)], perm=perm)
    want = HF.linear_block_fp8(x[T - 1:], *w)
    q, s = HF.quant_block_fp8(x[T - 1:])
    close(y, *(v.expand(2 * T, -1) for v in product64(q, s, *w)))
    close(want, *product64(q, s, *w))
    assert (y == y[0]).all()


def test_outputs_and_inputs_of_more_than_2_31_elements():
    from comfyui_amd import functional as HF
    g = gen(3)
    rows, K, N = 270000, 256, 8192
    w, sw = weight(g, N, K)
    x = tokens(g, rows, K)
    y = HF.linear_block_fp8(x, w, sw)
    part = slice(rows - 300, rows)
    q, s = HF.quant_block_fp8(x[part])
    close(y[part], *product64(q, s, w, sw))
    h, sh = HF.swiglu_block_fp8(x, w, sw, w, sw)
    close_cast(h[part], sh[part], q, s, w, sw, w, sw)
    del x, w
    # their cast rows as the next product's operand, read by the end of it
    w2, sw2 = weight(g, 128, N)
    z = HF.linear_block_fp8(h, w2, sw2, scale_x=sh)
    close(z[part], *product64(h[part], sh[part], w2, sw2))
    whole, scale = HF.quant_block_fp8(y)
    q, s = HF.quant_block_fp8(y[part])
    assert torch.equal(whole[part].view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale[part], s)


def test_two_graphs_in_turn():
    from comfyui_amd import functional as HF
    g = gen(5)
    K, H, E = 400, 528, 3
    up = [(*weight(g, H, K), *weight(g, H, K)) for _ in range(E)]
    down = [(*weight(g, K, H), None) for _ in range(E)]
    made = []
    for rows in (3, 120, 900):
        off = segments([rows - rows // 3, 0, rows // 3])

        def run(t, off=off):
            h, sh = HF.grouped_swiglu_block_fp8(t, off, up)
            return HF.grouped_linear_block_fp8(h, off, down, scale_a=sh)

        static = tokens(g, rows, K)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(static)
        made.append((graph, static, out, run, rows))
    for k in range(3):
        fresh = [tokens(gen(50 * k + m[4]), m[4], K) for m in made]
        for (graph, static, _, _, _), x in zip(made, fresh):
            static.copy_(x)
            graph.replay()
        want = [m[3](x) for m, x in zip(made, fresh)]
        torch.cuda.synchronize()
        for m, y in zip(made, want):
            assert torch.equal(m[2], y)


def test_views_of_larger_tensors():
    from comfyui_amd import functional as HF
    g = gen(8)
    w, sw = weight(g, 528, 272)
    bias = torch.randn(544, generator=g, device="cuda").bfloat16()
    x = tokens(g, 50, 272)
    part, rows = w[256:512], x[3:40]
    q, s = HF.quant_block_fp8(rows)
    y = HF.linear_block_fp8(rows, part, sw[2:4], bias=bias[8:264])
    close(y, *product64(q, s, part, sw[2:4], bias[8:264]))
    with pytest.raises(RuntimeError, match="16 bytes"):     # a bias that does not start on 16 bytes
        HF.linear_block_fp8(rows, part, sw[2:4], bias=bias[1:257])
    with pytest.raises(ValueError):                          # columns of a weight
        HF.linear_block_fp8(rows[:, :256].contiguous(), w[:, :256], sw[:, :2])
    with pytest.raises(ValueError):                          # scales of every other block
        HF.linear_block_fp8(rows, w[:256], sw[::2][:2])
    assert part.dtype == F8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,N", [(6, 272), (60, 784), (100, 272), (700, 1040), (4000, 3888)])
def test_a_row_that_is_not_finite_spoils_no_other(rows, N, dtype):
    from comfyui_amd import functional as HF
    g = gen(rows)
    K = 656
    x = tokens(g, rows, K, dtype)
    bad = [0, rows // 2, rows - 1]
    for r, (k, v) in zip(bad, ((5, float("inf")), (300, float("nan")), (655, float("-inf")))):
        x[r, k] = v
    fine = torch.ones(rows, dtype=torch.bool, device="cuda")
    fine[bad] = False
    w, w3 = weight(g, N, K), weight(g, N, K)
    y = HF.linear_block_fp8(x, *w)
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[fine]).all()
    h, sh = HF.swiglu_block_fp8(x, *w, *w3)
    values = h.float() * sh.repeat_interleave(128, 1)[:, :N]
    assert torch.isnan(values[bad]).all() and torch.isfinite(values[fine]).all()
    # NaN in a weight row: its feature everywhere, and its block of a cast row
    wn = w[0].clone()
    wn.view(torch.uint8)[130, 7] = 0x7F
    y = HF.linear_block_fp8(x, wn, w[1])
    assert torch.isnan(y[:, 130]).all() and torch.isfinite(y[fine][:, torch.arange(N, device="cuda") != 130]).all()
    h, sh = HF.swiglu_block_fp8(x, wn, w[1], *w3)
    values = h.float() * sh.repeat_interleave(128, 1)[:, :N]
    assert torch.isnan(values[:, 128:256]).all() and torch.isfinite(values[fine][:, :128]).all()


@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_both_ways_to_make_a_call_are_one(rows, dtype, monkeypatch):
    """The compiled calls against the ones made here: the same bytes, shapes, strides and refusals."""
    from comfyui_amd import functional as HF
    g = gen(rows)
    K, N, E = 656, 272, 3
    x = tokens(g, rows, K, dtype)
    q, s = HF.quant_block_fp8(x)
    bias = torch.randn(N, generator=g, device="cuda").to(dtype)
    experts = [(*weight(g, N, K), bias if e else None) for e in range(E)]
    up = [(*weight(g, N, K), *weight(g, N, K)) for _ in range(E)]
    off, off2 = segments([rows - rows // 2, 0, rows // 2]), segments([rows, 0, rows])
    perm = torch.randperm(2 * rows, generator=torch.Generator().manual_seed(rows)).to(torch.int32).cuda()
    w, sw, _ = experts[0]
    wide = (*weight(g, 400, K), *weight(g, 400, K))
    calls = [lambda: HF.quant_block_fp8(x), lambda: HF.quant_block_fp8(x.view(1, rows, K)), lambda: HF.linear_block_fp8(x, w, sw, bias=bias),
             lambda: HF.linear_block_fp8(q, w, sw, scale_x=s), lambda: HF.linear_block_fp8(q, w, sw, scale_x=s.contiguous(), out_dtype=dtype),
             lambda: HF.linear_block_fp8(x, w, sw, out_dtype=dtype), lambda: HF.grouped_linear_block_fp8(x, off, experts),
             lambda: HF.grouped_linear_block_fp8(q, off2, tuple(map(list, experts)), scale_a=s, perm=perm, out_dtype=dtype),
             lambda: HF.swiglu_block_fp8(x, *up[0]), lambda: HF.swiglu_block_fp8(q, *up[0], scale_x=s),
             lambda: HF.grouped_swiglu_block_fp8(x, off, up), lambda: HF.grouped_swiglu_block_fp8(q, off2, up, scale_a=s, perm=perm),
             lambda: HF.grouped_swiglu_block_fp8(x, off2, up, perm=perm, shared=wide), lambda: HF.grouped_swiglu_block_fp8(q, off, up, scale_a=s, shared=wide),
             lambda: HF.grouped_linear_block_fp8(x, off2, experts, perm=perm, shared=experts[1], a_static=x),
             lambda: HF.grouped_linear_block_fp8(q, off, experts, scale_a=s, shared=(*weight(gen(9), 400, 144), None), a_static=x[:, :144].contiguous(), out_dtype=dtype)]
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    refused = [lambda: HF.linear_block_fp8(x, w, sw, bias=bias.to(other)), lambda: HF.linear_block_fp8(x, w, sw, out_dtype=other),
               lambda: HF.linear_block_fp8(x, w, sw, scale_x=s), lambda: HF.linear_block_fp8(q, w, sw), lambda: HF.linear_block_fp8(x, w.cpu(), sw),
               lambda: HF.linear_block_fp8(x, w, sw[:1]), lambda: HF.linear_block_fp8(x[:, :K - 16], w, sw), lambda: HF.linear_block_fp8(x.float(), w, sw),
               lambda: HF.linear_block_fp8(x, w.float(), sw), lambda: HF.linear_block_fp8(x, w, sw.double()), lambda: HF.linear_block_fp8(x, w[:-8], sw),
               lambda: HF.grouped_linear_block_fp8(x, off.long(), experts), lambda: HF.grouped_linear_block_fp8(x, off[:-1], experts),
               lambda: HF.grouped_linear_block_fp8(x, off, []), lambda: HF.grouped_linear_block_fp8(x, off2, experts, perm=perm[:-1]),
               lambda: HF.grouped_linear_block_fp8(x, off, experts[:2] + [(experts[2][0][:-16], experts[2][1], None)]),
               lambda: HF.grouped_swiglu_block_fp8(x, off, up[:2] + [(*up[2][:2], up[2][2][:, :-16], up[2][3])]),
               lambda: HF.swiglu_block_fp8(x[None], *up[0]), lambda: HF.quant_block_fp8(x.t()), lambda: HF.quant_block_fp8(x[:, :24].contiguous())]

    def outcome(f):
        try:
            f()
        except Exception as e:  # noqa: BLE001
            return type(e), str(e)
        return None

    refused += [lambda: HF.grouped_swiglu_block_fp8(x, off, up, shared=up[0][:3]), lambda: HF.grouped_linear_block_fp8(x, off, experts, shared=experts[0]),
                lambda: HF.grouped_linear_block_fp8(q, off, experts, scale_a=s, shared=experts[0], a_static=q),
                lambda: HF.grouped_swiglu_block_fp8(x, off, up, shared=(*up[0][:2], up[0][2][:-16], up[0][3]))]
    made, no = [f() for f in calls], [outcome(f) for f in refused]
    with monkeypatch.context() as m:
        m.setattr(HF, "_stream_here", lambda t: None)
        slow, slow_no = [f() for f in calls], [outcome(f) for f in refused]
    for a, b in zip(made, slow):
        for t, u in zip(*((v if isinstance(v, tuple) else (v,)) for v in (a, b))):
            assert t.dtype == u.dtype and t.shape == u.shape and t.stride() == u.stride()
            assert torch.equal(t.contiguous().view(torch.uint8), u.contiguous().view(torch.uint8))
    assert no == slow_no and all(n is not None for n in no)


def test_threads():
    """Calls from several Python threads on streams of their own."""
    import threading

    from comfyui_amd import functional as HF
    g = gen(4)
    xs = [tokens(g, rows, 656) for rows in (2, 50, 300, 7)]
    up = [(*weight(g, 272, 656), *weight(g, 272, 656)) for _ in range(2)]
    w, sw = weight(g, 400, 272)

    def run(x):
        n = x.shape[0]
        h, sh = HF.grouped_swiglu_block_fp8(x, off[n], up)
        return HF.linear_block_fp8(h, w, sw, scale_x=sh)

    off = {x.shape[0]: segments([x.shape[0] // 2, x.shape[0] - x.shape[0] // 2]) for x in xs}
    want = [run(x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [run(xs[i]) for _ in range(30)]
            torch.cuda.current_stream().synchronize()
        if not all(torch.equal(y, want[i]) for y in got):
            bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
