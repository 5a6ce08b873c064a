"""Layer norm, its gradients and those of the modulated norm against 64 bits (tests/norm64.py derives the tolerances)."""
import pytest
import torch

from tests import norm64
from tests.norm64 import close

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_of(g, shape, dtype, offset=0.3):
    channel = torch.exp(0.7 * torch.randn(shape[-1], generator=g, device="cuda"))
    return ((torch.randn(shape, generator=g, device="cuda") + offset) * channel).to(dtype)


def gains(g, D, dtype):
    return ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype), torch.randn(D, generator=g, device="cuda").to(dtype))


def check(x, w, b, dy, eps):
    from comfyui_amd import functional as HF
    y = HF.layer_norm(x, w, b, eps=eps)
    dx, dw, db = HF.layer_norm_backward(dy, x, w, b, eps=eps)
    x2, dy2 = x.reshape(-1, x.shape[-1]), dy.reshape(-1, x.shape[-1])
    close(y.reshape(x2.shape), *norm64.norm(x2, w, b, eps), "y")
    (e, ee), (ew, eew), (eb, eeb) = norm64.backward(dy2, x2, 1.0 if w is None else w.double(), eps)
    close(dx.reshape(x2.shape), e, ee, "dx")
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    if w is not None:
        close(dw, ew, eew, "dw")
    if b is not None:
        close(db, eb, eeb, "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (1, 7), (5, 64), (17, 511), (9, 512), (33, 520), (1000, 1024), (77, 1153), (65, 2048), (300, 2560),
                                    (7, 2561), (130, 3584), (19, 4096), (11, 4100), (600, 6912), (2, 8192), (3, 8193), (5, 16384), (2100, 96)])
def test_sizes(dtype, rows, D):
    g = gen(rows * 7 + D)
    x = rows_of(g, (rows, D), dtype)
    w, b = gains(g, D, dtype)
    check(x, w, b, torch.randn((rows, D), generator=g, device="cuda").to(dtype), 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_w,with_b,gain_type", [(False, False, None), (True, False, None), (False, True, None), (True, True, torch.float32),
                                                     (False, True, torch.float32)])
def test_gains(dtype, with_w, with_b, gain_type):
    g = gen(5)
    x = rows_of(g, (3, 41, 640), dtype)
    w, b = gains(g, 640, gain_type or dtype)
    check(x, w if with_w else None, b if with_b else None, torch.randn(x.shape, generator=g, device="cuda").to(dtype), 1e-6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,D", [(1, 1, 256), (3, 5, 264), (2, 700, 2560), (300, 3, 96), (600, 40, 64), (5, 333, 1100), (2, 50, 5000)])
def test_modulated(dtype, B, L, D):
    from comfyui_amd import functional as HF
    g = gen(B * 100 + L)
    x = rows_of(g, (B * L, D), dtype)
    dy = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
    scale = (0.4 * torch.randn((B, 1, D), generator=g, device="cuda")).to(dtype)
    dx, ds, dsh = HF.ln_modulate_backward(dy, x, scale, L, eps=1e-6)
    (e, ee), (es, ees), (eb, eeb) = norm64.backward(dy.view(B, L, D), x.view(B, L, D), 1 + scale.double(), 1e-6, rows_dim=1)
    close(dx.view(B, L, D), e, ee, "dx")
    close(ds, es, ees, "dscale")
    close(dsh, eb, eeb, "dshift")


def test_gradient_of_the_modulated_forward():
    """What ln_modulate's results move by where scale and shift grow by 1, in which they are linear, is what the gradients tell. ln_modulate rounds
    the normed value, 1 + scale, their product and the sum to bf16: 2^-8 of the product three times and of the sum once."""
    from comfyui_amd import functional as HF
    g = gen(11)
    B, L, D = 2, 64, 512
    x = rows_of(g, (B * L, D), torch.bfloat16)
    scale, shift = ((0.4 * torch.randn((B, D), generator=g, device="cuda")).bfloat16() for _ in range(2))
    bump = torch.randint(0, 2, (B, D), generator=g, device="cuda").bfloat16()
    n = norm64.stats(x, 1e-6)[0].view(B, L, D)
    dy = torch.sign((n + 1) * bump[:, None]).reshape(x.shape).bfloat16()     # nothing cancels in the sum
    _, ds, dsh = HF.ln_modulate_backward(dy, x, scale, L)
    told = ((ds.double() + dsh.double()) * bump).sum()
    moved, room = 0.0, 2.0 ** -8 * ((ds.double().abs() + dsh.double().abs()) * bump).sum()
    for sign, sc, sh in ((-1, scale, shift), (1, scale + bump, shift + bump)):
        y = HF.ln_modulate(x, sc, sh, L).double().view(B, L, D)
        moved = moved + sign * (y * dy.view(B, L, D)).sum()
        room = room + (2.0 ** -8 * (3 * (n * (1 + sc.double()[:, None])).abs() + y.abs()) * dy.view(B, L, D).abs()).sum()
        room = room + (2.0 ** -8 * (sc.double().abs() + sh.double().abs()) * (n.abs().sum(1) + L)).sum()   # the sums scale + 1, shift + 1 in bf16
    assert abs(moved - told) < room and told > 3 * room


@pytest.mark.parametrize("dtype", TYPES)
def test_views_off_their_alignment(dtype):
    g = gen(3)
    flat = rows_of(g, (41 * 515 + 3,), dtype)
    x = flat[3:].view(41, 515)
    w, b = (rows_of(g, (516,), dtype)[1:] for _ in range(2))
    dy = torch.randn((41 * 515 + 1,), generator=g, device="cuda").to(dtype)[1:].view(41, 515)
    check(x, w, b, dy, 1e-5)


@pytest.mark.parametrize("D", [96, 2560, 5000])
def test_a_bad_row_stays_its_own(D):
    from comfyui_amd import functional as HF
    g = gen(D)
    x = rows_of(g, (60, D), torch.bfloat16)
    dy = torch.randn(x.shape, generator=g, device="cuda").bfloat16()
    w, b = gains(g, D, torch.bfloat16)
    y, (dx, _, db) = HF.layer_norm(x, w, b), HF.layer_norm_backward(dy, x, w, b)
    bad = x.clone()
    bad[7, 3], bad[20, D - 1] = float("nan"), float("inf")
    y2, (dx2, _, db2) = HF.layer_norm(bad, w, b), HF.layer_norm_backward(dy, bad, w, b)
    ok = torch.ones(60, dtype=torch.bool, device="cuda")
    ok[[7, 20]] = False
    assert torch.equal(y[ok], y2[ok]) and torch.equal(dx[ok], dx2[ok]) and torch.equal(db, db2)
    assert y2[~ok].isnan().all() and dx2[~ok].isnan().all()


def test_equal_values_and_large_offsets():
    g = gen(2)
    for dtype in TYPES:
        x = torch.full((5, 2560), 3.0, device="cuda", dtype=dtype)
        w, b = gains(g, 2560, dtype)
        dy = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
        check(x, w, b, dy, 1e-5)                       # a variance of 0
    x = (torch.randn((50, 2560), generator=g, device="cuda") + 4096.0)   # cancels in a variance of squares
    check(x, *gains(g, 2560, torch.float32), torch.randn(x.shape, generator=g, device="cuda"), 1e-5)


def test_no_rows():
    from comfyui_amd import functional as HF
    for dtype in TYPES:
        x = torch.empty((0, 640), device="cuda", dtype=dtype)
        w, b = gains(gen(1), 640, dtype)
        assert HF.layer_norm(x, w, b).shape == x.shape
        dx, dw, db = HF.layer_norm_backward(x, x, w, b)
        assert dx.shape == x.shape and not dw.any() and not db.any()
        dx, ds, dsh = HF.ln_modulate_backward(x, x, x, 5)
        assert ds.shape == (0, 640) and dsh.shape == (0, 640)


def test_refused_on_the_device():
    from comfyui_amd import functional as HF
    x = torch.zeros((8, 64), device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(64, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: HF.layer_norm(x[:, ::2]), lambda: HF.layer_norm(x, w[:32]), lambda: HF.layer_norm(x, w.cpu()),
                 lambda: HF.layer_norm(torch.zeros((2, 16385), device="cuda")), lambda: HF.layer_norm(x[:, :0]),
                 lambda: HF.layer_norm(torch.zeros((), device="cuda")), lambda: HF.layer_norm_backward(x[:4], x, w, w),
                 lambda: HF.layer_norm_backward(x.float(), x, w, w), lambda: HF.ln_modulate_backward(x, x, w[None], 3),
                 lambda: HF.ln_modulate_backward(x, x, w, 8), lambda: HF.ln_modulate_backward(x[None], x[None], w[None], 8)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: HF.layer_norm(x, w.half()), lambda: HF.layer_norm(x, w, w.float())):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("rows", [12, 3000])
def test_captured_replayed_and_on_another_stream(rows):
    """Two graphs with workspaces of their own, replayed in turn with eager work between, on inputs written anew."""
    from comfyui_amd import functional as HF
    g = gen(rows)
    sets = []
    for D in (640, 2560):
        x = rows_of(g, (rows, D), torch.bfloat16)
        w, b = gains(g, D, torch.bfloat16)
        sets.append([x, w, b, torch.randn(x.shape, generator=g, device="cuda").bfloat16()])
    def call(s):
        return (HF.layer_norm(s[0], s[1], s[2]), *HF.layer_norm_backward(s[3], s[0], s[1], s[2]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        elsewhere = [call(s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    for s, got in zip(sets, elsewhere):
        assert all(torch.equal(a, c) for a, c in zip(call(s), got))
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(s))
        graphs.append(graph)
    for turn in range(3):
        for s in sets:
            s[0].copy_(rows_of(g, s[0].shape, torch.bfloat16))
        for graph in graphs:
            graph.replay()
        for s, out in zip(sets, outs):
            assert all(torch.equal(a, c) for a, c in zip(call(s), out)), turn
        torch.cuda.synchronize()
