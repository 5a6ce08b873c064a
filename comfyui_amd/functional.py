"""Tensor-level wrappers over the C ABI: they check devices/dtypes/shapes, allocate
outputs with torch (device memory and stream plumbing only) and enqueue the HIP
kernels on torch's current stream. Nothing here computes with torch.
"""
import contextlib
import ctypes
import logging

import torch

from . import _lib
from ._lib import FfnWeights, LayerArgs, LayerLayout, W_BF16, W_E4M3FN, check, lib, ptr

try:
    from . import _block_calls
    if (getattr(_block_calls, "torch_version", None), getattr(_block_calls, "hdmoe_version", None)) != (torch.__version__, lib.hdmoe_version()):
        raise ImportError(f"not built for torch {torch.__version__} and this library")
except ImportError as e:   # host code only: every call it makes is made below as well, at a few times the host's time
    logging.warning("comfyui_amd: no compiled calls of the block-scaled operators (%s). `python -m comfyui_amd.build` builds them.", e)
    _block_calls = None

try:
    from . import _row_calls
    if (getattr(_row_calls, "torch_version", None), getattr(_row_calls, "hdmoe_version", None)) != (torch.__version__, lib.hdmoe_version()):
        raise ImportError(f"not built for torch {torch.__version__} and this library")
except ImportError as e:   # as above
    logging.warning("comfyui_amd: no compiled calls of the layer norm, the balance loss and the adapters (%s). `python -m comfyui_amd.build` builds them.", e)
    _row_calls = None

FP8 = torch.float8_e4m3fn
BF16 = torch.bfloat16
F16 = torch.float16
FP8_UPCAST = "float8_e4m3fn multiplied in bfloat16"   # a "weight dtype" of moe_ffn / ffn_swiglu: no activation is cast
TOPK = _lib.TOPK
ACT_DTYPES = (BF16, F16)   # 16-bit activation formats; fp16 is served by the *_f16 entry points (Hunyuan3D block)


def _act_dtype(t, what):
    """The tensor's dtype if it is one of the two 16-bit activation formats."""
    if t.dtype not in ACT_DTYPES:
        raise TypeError(f"{what}: expected bfloat16 or float16, got {t.dtype}")
    return t.dtype


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _need_hip(t, what, dtype=None):
    if not t.is_cuda:
        raise RuntimeError(f"{what}: tensor is on {t.device}; comfyui_amd only computes on a HIP device "
                           "(there is no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: tensor must be contiguous")


def weight_dtype_code(dtype):
    if dtype == BF16:
        return W_BF16
    if dtype == FP8:
        return W_E4M3FN
    if dtype == FP8_UPCAST:
        return _lib.W_E4M3FN_UPCAST
    if dtype == F16:
        return _lib.W_F16      # hdmoe_linear_bias only
    raise TypeError(f"unsupported weight dtype {dtype}: the HIP path takes bfloat16 or float8_e4m3fn weights")


def moe_ffn_rows_fit(T, D, H, Hs):
    """Whether hdmoe_moe_ffn takes this many tokens with 16-bit activations (4 GiB per operand, 2 GiB for the tokens that it reads
    through the permutation)."""
    return max(3 * T * D, 2 * T * H, T * Hs) * 2 < 2 ** 32 and T * D * 2 < 2 ** 31


def gate_top2(x2d, gate_w):
    """MoEGate scoring + top-2 on the device. x2d [T,D] bf16 (or fp16), gate_w [E,D] of the same dtype
    -> topk_idx int32 [T,2], topk_weight [T,2] of that dtype."""
    dt = _act_dtype(x2d, "gate_top2 x")
    _need_hip(x2d, "gate_top2 x", dt)
    _need_hip(gate_w, "gate_top2 gate weight", dt)
    T, D = x2d.shape
    E = gate_w.shape[0]
    if gate_w.shape[1] != D:
        raise ValueError(f"gate weight {tuple(gate_w.shape)} does not match hidden size {D}")
    idx = torch.empty((T, 2), dtype=torch.int32, device=x2d.device)
    w = torch.empty((T, 2), dtype=dt, device=x2d.device)
    fn = lib.hdmoe_gate_top2 if dt == BF16 else lib.hdmoe_gate_top2_f16
    check(fn(ptr(x2d), ptr(gate_w), T, D, E, ptr(idx), ptr(w), _stream(x2d)))
    return idx, w


def renorm_top2(topk_weight):
    """topk_weight / (topk_weight.sum(-1, keepdim=True) + 1e-20) for the [T, 2] bf16 gate weights."""
    _need_hip(topk_weight, "renorm_top2 topk_weight", BF16)
    if topk_weight.dim() != 2 or topk_weight.shape[1] != 2 or not topk_weight.is_contiguous():
        raise ValueError("renorm_top2: expected a contiguous [T, 2] tensor")
    out = torch.empty_like(topk_weight)
    if topk_weight.shape[0] == 0:
        return out
    check(lib.hdmoe_renorm_top2_bf16(ptr(topk_weight), topk_weight.shape[0], ptr(out), _stream(topk_weight)))
    return out


def dispatch(topk_idx, E):
    """Stable permutation of the flat slots by expert.
    -> counts [E], offsets [E+1], perm [2T], inv_perm [2T] (int32, device)."""
    _need_hip(topk_idx, "dispatch topk_idx", torch.int32)
    T = topk_idx.shape[0]
    dev = topk_idx.device
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(2 * T, dtype=torch.int32, device=dev)
    inv = torch.empty(2 * T, dtype=torch.int32, device=dev)
    nbytes = lib.hdmoe_dispatch_workspace_bytes(T, E)
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
    check(lib.hdmoe_dispatch(ptr(topk_idx), T, E, ptr(counts), ptr(offsets), ptr(perm), ptr(inv), ptr(ws), nbytes,
                             _stream(topk_idx)))
    return counts, offsets, perm, inv


def _scale_ptr(s, device, what):
    if s is None:
        return None
    if s.device != device or s.dtype != torch.float32 or s.numel() != 1:
        raise ValueError(f"{what} must be an fp32 scalar tensor on {device}")
    return s.data_ptr()


def quant_fp8(x, scale_input):
    """fp8_linear's activation cast: x bf16 [..., D] -> float8_e4m3fn, same shape."""
    _need_hip(x, "quant_fp8 x", BF16)
    D = x.shape[-1]
    out = torch.empty(x.shape, dtype=FP8, device=x.device)
    check(lib.hdmoe_quant_fp8(ptr(x), x.numel() // D, D, _scale_ptr(scale_input, x.device, "scale_input"), ptr(out),
                              _stream(x)))
    return out


def quant_permute_fp8(x2d, perm, offsets, scale_inputs):
    """Gather rows by perm and quantise each with its expert's scale_input. -> [2T,D] fp8."""
    _need_hip(x2d, "quant_permute_fp8 x", BF16)
    T, D = x2d.shape
    E = len(scale_inputs)
    arr = (ctypes.c_void_p * E)(*[_scale_ptr(s, x2d.device, "scale_input") for s in scale_inputs])
    out = torch.empty((2 * T, D), dtype=FP8, device=x2d.device)
    check(lib.hdmoe_quant_permute_fp8(ptr(x2d), ptr(perm), ptr(offsets), T, D, E, arr, ptr(out), _stream(x2d)))
    return out


def permute_bf16(x2d, perm):
    """a[r] = x[perm[r] / 2]; rows are copied as bytes, so fp16 rows go through the same kernel."""
    dt = _act_dtype(x2d, "permute_bf16 x")
    _need_hip(x2d, "permute_bf16 x", dt)
    T, D = x2d.shape
    out = torch.empty((2 * T, D), dtype=dt, device=x2d.device)
    check(lib.hdmoe_permute_bf16(ptr(x2d), ptr(perm), T, D, ptr(out), _stream(x2d)))
    return out


def _linear_groups(dt, weight_code, K, N, act, device, experts=(), a=None, perm=None, offsets=None, rows=0, out=None,
                   shared=None, a_static=None, out_static=None, fixed_k_cut=False):
    """hdmoe_linear_groups with its working memory. experts: list of LinearGroup; shared: LinearGroup or None."""
    args = _lib.LinearArgs()
    args.act_dtype = W_BF16 if dt == BF16 else _lib.W_F16
    args.weight_dtype = args.act_dtype if weight_code is None else weight_code
    args.K, args.N, args.act, args.fixed_k_cut = K, N, act, 1 if fixed_k_cut else 0
    if len(experts) > 0 and rows > 0:
        args.E, args.rows = len(experts), rows
        arr = (_lib.LinearGroup * len(experts))(*experts)
        args.a, args.offsets, args.experts, args.out = ptr(a), ptr(offsets), arr, ptr(out)
        if perm is not None:
            args.perm, args.T = ptr(perm), a.shape[0]
    if shared is not None and a_static.shape[0] > 0:
        args.a_static, args.shared, args.out_static = ptr(a_static), ctypes.pointer(shared), ptr(out_static)
        args.rows_static = a_static.shape[0]
    if args.rows == 0 and args.rows_static == 0:
        return
    ref = ctypes.byref(args)
    nbytes = lib.hdmoe_linear_groups_workspace_bytes(ref)
    if nbytes > 0:   # 0: nothing of it would be used, or sizes the call below refuses
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    check(lib.hdmoe_linear_groups(ref, torch.cuda.current_stream(device).cuda_stream))


def _linear_group(weight, bias, K, N, what, dtype=BF16):
    _need_hip(weight, f"{what} weight", dtype)
    if tuple(weight.shape) != (N, K):
        raise ValueError(f"{what}: weight shape {tuple(weight.shape)} != ({N}, {K})")
    g = _lib.LinearGroup()
    g.weight = ptr(weight)
    if bias is not None:
        _need_hip(bias, f"{what} bias", dtype)
        if tuple(bias.shape) != (N,):
            raise ValueError(f"{what}: bias shape {tuple(bias.shape)} != ({N},)")
        g.bias = ptr(bias)
    return g


def linear(a2d, weight, scale_weight=None, scale_input=None, bias=None, fixed_k_cut=False):
    """a2d [rows,K] (fp8 for fp8 weights, bf16 for bf16 weights, fp16 for fp16 weights) x weight [N,K]^T (+ bias [N])
    -> [rows,N] bf16 (fp16 for fp16 weights); the bias joins the fp32 result before the one rounding.
    fixed_k_cut: see grouped_linear (16-bit activations; with fp8 ones a row never depends on the number of rows)."""
    code = weight_dtype_code(weight.dtype)
    _need_hip(a2d, "linear activations", weight.dtype)
    _need_hip(weight, "linear weight")
    rows, K = a2d.shape
    N = weight.shape[0]
    if weight.shape[1] != K:
        raise ValueError(f"linear: activations [{rows},{K}] do not match weight {tuple(weight.shape)}")
    out_dtype = F16 if weight.dtype == F16 else BF16
    if bias is not None:
        _need_hip(bias, "linear bias", out_dtype)
        if bias.shape != (N,) or not bias.is_contiguous():
            raise ValueError(f"linear: bias {tuple(bias.shape)} does not match {N} output features")
    out = torch.empty((rows, N), dtype=out_dtype, device=a2d.device)
    if code != W_E4M3FN:
        g = _lib.LinearGroup(ptr(weight), ptr(bias), None)
        _linear_groups(out_dtype, None, K, N, _lib.ACT_NONE, a2d.device, shared=g, a_static=a2d, out_static=out,
                       fixed_k_cut=fixed_k_cut)
        return out
    check(lib.hdmoe_linear_bias(code, ptr(a2d), rows, K, N, ptr(weight),
                                _scale_ptr(scale_weight, a2d.device, "scale_weight"),
                                _scale_ptr(scale_input, a2d.device, "scale_input"), ptr(bias), ptr(out), _stream(a2d)))
    return out


def linear_upcast_fits(K, N):
    """Whether a Linear of these sizes has a kernel that multiplies its fp8 weight in bf16."""
    return K % 128 == 0 and K >= 384 and N % 256 == 0


def linear_upcast_aligned(*tensors):
    """Whether that kernel may read these as they lie: it loads 16 bytes at a time straight into LDS. (What is not contiguous is
    copied first, to an aligned place.)"""
    return all(t.data_ptr() % 16 == 0 or not t.is_contiguous() for t in tensors)


def linear_upcast(a2d, weight, scale=None, bias=None, fixed_k_cut=False):
    """bf16( (a2d . weight^T) * bf16(scale) + bias ) for bf16 a2d [rows,K] and a float8_e4m3fn weight [N,K]: the Linear
    without fp8 matrix multiply on the stored bytes (linear_upcast_fits sizes)."""
    _need_hip(a2d, "linear_upcast activations", BF16)
    _need_hip(weight, "linear_upcast weight", FP8)
    rows, K = a2d.shape
    N = weight.shape[0]
    if weight.shape[1] != K:
        raise ValueError(f"linear_upcast: activations [{rows},{K}] do not match weight {tuple(weight.shape)}")
    if bias is not None:
        _need_hip(bias, "linear_upcast bias", BF16)
        if bias.shape != (N,):
            raise ValueError(f"linear_upcast: bias {tuple(bias.shape)} does not match {N} output features")
    if not linear_upcast_aligned(a2d, weight):
        raise ValueError("linear_upcast: activations and weight must start on a multiple of 16 bytes")
    if bias is not None and bias.data_ptr() % 8 != 0:
        bias = bias.clone()
    out = torch.empty((rows, N), dtype=BF16, device=a2d.device)
    g = _lib.LinearGroup(ptr(weight), ptr(bias), _scale_ptr(scale, a2d.device, "linear_upcast scale"))
    _linear_groups(BF16, _lib.W_E4M3FN_UPCAST, K, N, _lib.ACT_NONE, a2d.device, shared=g, a_static=a2d, out_static=out,
                   fixed_k_cut=fixed_k_cut)
    return out


def silu_mul(a, b):
    _need_hip(a, "silu_mul a", BF16)
    _need_hip(b, "silu_mul b", BF16)
    if a.shape != b.shape:
        raise ValueError("silu_mul: shape mismatch")
    out = torch.empty_like(a)
    check(lib.hdmoe_silu_mul_bf16(ptr(a), ptr(b), a.numel(), ptr(out), _stream(a)))
    return out


def gelu(x):
    """F.gelu (erf form) of a contiguous bf16 or fp16 tensor."""
    dt = _act_dtype(x, "gelu x")
    _need_hip(x, "gelu x", dt)
    out = torch.empty_like(x)
    fn = lib.hdmoe_gelu_bf16 if dt == BF16 else lib.hdmoe_gelu_f16
    check(fn(ptr(x), x.numel(), ptr(out), _stream(x)))
    return out


def scale_to_bf16(src, scale):
    """bf16(bf16(src) * bf16(scale)) for src in fp8 or bf16."""
    code = weight_dtype_code(src.dtype)
    _need_hip(src, "scale_to_bf16 src")
    out = torch.empty(src.shape, dtype=BF16, device=src.device)
    check(lib.hdmoe_scale_to_bf16(code, ptr(src), src.numel(), _scale_ptr(scale, src.device, "scale"), ptr(out),
                                  _stream(src)))
    return out


def combine(y_sorted, inv_perm, topk_weight, shared):
    dt = _act_dtype(y_sorted, "combine y")
    _need_hip(y_sorted, "combine y", dt)
    _need_hip(topk_weight, "combine topk_weight", dt)
    if shared is not None:
        _need_hip(shared, "combine shared", dt)
    T = topk_weight.shape[0]
    D = y_sorted.shape[1]
    out = torch.empty((T, D), dtype=dt, device=y_sorted.device)
    fn = lib.hdmoe_combine if dt == BF16 else lib.hdmoe_combine_f16
    check(fn(ptr(y_sorted), ptr(inv_perm), ptr(topk_weight), ptr(shared), T, D, ptr(out), _stream(y_sorted)))
    return out


def grouped_linear(a_sorted, offsets, experts, a_static=None, shared=None, act="none", fixed_k_cut=False):
    """Linear (+ bias, + erf GELU) of every expert over its row segment of `a_sorted` [rows, K] and, optionally, of
    one more (weight, bias) over all rows of `a_static`, in one launch. experts: list of (weight [N,K], bias [N] or
    None). Returns (out_sorted [rows, N], out_static [rows_static, N] or None).
    fixed_k_cut: no tile of the last round is cut along K, which otherwise goes by the segment sizes: a row's bytes then do not
    depend on the other rows."""
    code = {"none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU}[act]
    dt = _act_dtype(a_sorted, "grouped_linear a")   # bf16, or fp16 throughout
    _need_hip(a_sorted, "grouped_linear a", dt)
    rows, K = a_sorted.shape
    N = experts[0][0].shape[0] if experts else shared[0].shape[0]
    groups = [_linear_group(w, b, K, N, f"grouped_linear expert {i}", dt) for i, (w, b) in enumerate(experts)]
    out = torch.empty((rows, N), dtype=dt, device=a_sorted.device)
    out_static, sh = None, None
    if shared is not None:
        _need_hip(a_static, "grouped_linear a_static", dt)
        sh = _linear_group(shared[0], shared[1], K, N, "grouped_linear shared", dt)
        out_static = torch.empty((a_static.shape[0], N), dtype=dt, device=a_sorted.device)
    _linear_groups(dt, None, K, N, code, a_sorted.device, groups, a_sorted, None, offsets, rows, out, sh, a_static, out_static,
                   fixed_k_cut)
    return out, out_static


def grouped_linear_tokens(x2d, perm, offsets, experts, shared=None, act="none", fixed_k_cut=False):
    """The first Linear (+ bias, + erf GELU) of every expert on the rows of `x2d` [T, K] its segment selects through
    the dispatch permutation (sorted row r = token perm[r] // 2; nothing is copied into expert order), and of
    `shared` (weight, bias) on all T rows, in one launch. Returns (out_sorted [2T, N], out_shared [T, N] or None)."""
    code = {"none": _lib.ACT_NONE, "gelu": _lib.ACT_GELU}[act]
    dt = _act_dtype(x2d, "grouped_linear_tokens x")
    _need_hip(x2d, "grouped_linear_tokens x", dt)
    T, K = x2d.shape
    N = experts[0][0].shape[0]
    groups = [_linear_group(w, b, K, N, f"grouped_linear_tokens expert {i}", dt) for i, (w, b) in enumerate(experts)]
    out = torch.empty((T * _lib.TOPK, N), dtype=dt, device=x2d.device)
    out_shared, sh = None, None
    if shared is not None:
        sh = _linear_group(shared[0], shared[1], K, N, "grouped_linear_tokens shared", dt)
        out_shared = torch.empty((T, N), dtype=dt, device=x2d.device)
    _linear_groups(dt, None, K, N, code, x2d.device, groups, x2d, perm, offsets, T * _lib.TOPK, out, sh, x2d, out_shared,
                   fixed_k_cut)
    return out, out_shared


def stochastic_round_e4m3fn(weight, scale=None, seed=0, out=None):
    """weight (fp32 or bf16, HIP) / scale (fp32 scalar tensor or None) -> float8_e4m3fn by stochastic rounding
    (comfy/float.py:14-67 behind comfy/ops.py:419-426), one kernel. `out`: a contiguous float8_e4m3fn tensor of the
    weight's shape, of other memory than the weight's and starting on 4 bytes, that takes the result."""
    _need_hip(weight, "stochastic_round_e4m3fn weight")
    if weight.dtype == torch.float32:
        code = _lib.SRC_F32
    elif weight.dtype == BF16:
        code = _lib.SRC_BF16
    else:
        raise TypeError(f"stochastic_round_e4m3fn: expected float32 or bfloat16, got {weight.dtype}")
    if out is None:
        out = torch.empty(weight.shape, dtype=FP8, device=weight.device)
    else:
        _need_hip(out, "stochastic_round_e4m3fn out", FP8)
        if out.shape != weight.shape or out.device != weight.device:
            raise ValueError(f"stochastic_round_e4m3fn: out {tuple(out.shape)} on {out.device} for a weight "
                             f"{tuple(weight.shape)} on {weight.device}")
    check(lib.hdmoe_stochastic_round_e4m3fn(code, ptr(weight), weight.numel(),
                                            _scale_ptr(scale, weight.device, "stochastic_round_e4m3fn scale"),
                                            int(seed) & 0xFFFFFFFFFFFFFFFF, ptr(out), _stream(weight)))
    return out


def _per_batch(t, what, D, device):
    """[B, D] (or [B, 1, D]) bf16 modulation rows -> contiguous [B, D]."""
    _need_hip(t, what, BF16)
    if t.dim() == 3 and t.shape[1] == 1:
        t = t[:, 0]
    if t.dim() != 2 or t.shape[1] != D or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous [batch, {D}] tensor, got {tuple(t.shape)}")
    return t


def ln_modulate(x2d, scale, shift, tokens_per_batch, eps=1e-6):
    """bf16 LayerNorm(x) * (1 + scale) + shift with scale/shift one row per batch item
    (comfy/ldm/hidream/model.py:430-431, 516-517)."""
    _need_hip(x2d, "ln_modulate x", BF16)
    T, D = x2d.shape
    scale = _per_batch(scale, "ln_modulate scale", D, x2d.device)
    shift = _per_batch(shift, "ln_modulate shift", D, x2d.device)
    if tokens_per_batch <= 0 or T != scale.shape[0] * tokens_per_batch or shift.shape != scale.shape:
        raise ValueError(f"ln_modulate: T={T} is not batch={scale.shape[0]} x tokens_per_batch={tokens_per_batch}")
    out = torch.empty_like(x2d)
    check(lib.hdmoe_ln_modulate_bf16(ptr(x2d), ptr(scale), ptr(shift), T, D, tokens_per_batch, eps, ptr(out),
                                     _stream(x2d)))
    return out


def combine_gated_residual(y_sorted, inv_perm, topk_weight, shared, gate, residual, tokens_per_batch):
    """combine(), then gate * y + residual (comfy/ldm/hidream/model.py:432-433, 518-523)."""
    _need_hip(y_sorted, "combine y", BF16)
    _need_hip(topk_weight, "combine topk_weight", BF16)
    _need_hip(residual, "combine residual", BF16)
    T = topk_weight.shape[0]
    D = y_sorted.shape[1]
    gate = _per_batch(gate, "combine gate", D, y_sorted.device)
    if tokens_per_batch <= 0 or T != gate.shape[0] * tokens_per_batch or tuple(residual.shape) != (T, D):
        raise ValueError(f"combine_gated_residual: T={T}, batch={gate.shape[0]}, tokens_per_batch={tokens_per_batch}")
    out = torch.empty((T, D), dtype=BF16, device=y_sorted.device)
    check(lib.hdmoe_combine_gated_residual(ptr(y_sorted), ptr(inv_perm), ptr(topk_weight), ptr(shared), ptr(gate),
                                           ptr(residual), tokens_per_batch, T, D, ptr(out), _stream(y_sorted)))
    return out


def gated_residual(y2d, gate, residual2d, tokens_per_batch):
    """gate * y + residual behind a dense feed-forward (comfy/ldm/hidream/model.py:519-523)."""
    _need_hip(y2d, "gated_residual y", BF16)
    _need_hip(residual2d, "gated_residual residual", BF16)
    T, D = y2d.shape
    gate = _per_batch(gate, "gated_residual gate", D, y2d.device)
    if tokens_per_batch <= 0 or T != gate.shape[0] * tokens_per_batch or tuple(residual2d.shape) != (T, D):
        raise ValueError(f"gated_residual: T={T}, batch={gate.shape[0]}, tokens_per_batch={tokens_per_batch}")
    out = torch.empty_like(y2d)
    check(lib.hdmoe_gated_residual_bf16(ptr(y2d), ptr(gate), ptr(residual2d), tokens_per_batch, T, D, ptr(out),
                                        _stream(y2d)))
    return out


def make_ffn_weights(w1, w2, w3, scales=None, same_scale_in13=False):
    """Fill an hdmoe_ffn_weights. scales: dict with optional fp32 scalar tensors
    scale_w1/2/3 and scale_in1/2/3 (fp8 only). same_scale_in13: the caller has checked that scale_in1 and
    scale_in3, two different tensors, hold the same value (the library refuses two different pointers otherwise)."""
    fw = FfnWeights()
    fw.w1, fw.w2, fw.w3 = ptr(w1), ptr(w2), ptr(w3)
    if scales:
        for k, v in scales.items():
            setattr(fw, k, ptr(v))
    fw.same_scale_in13 = 1 if same_scale_in13 else 0
    return fw


def grouped_swiglu(a, offsets, experts, H):
    """experts: list of FfnWeights. a [2T,D] -> h [2T,H] (same element type as a)."""
    code = weight_dtype_code(a.dtype)
    _need_hip(a, "grouped_swiglu a")
    rows, D = a.shape
    E = len(experts)
    arr = (FfnWeights * E)(*experts)
    h = torch.empty((rows, H), dtype=a.dtype, device=a.device)
    check(lib.hdmoe_grouped_swiglu(code, ptr(a), ptr(offsets), rows, E, D, H, arr, ptr(h), _stream(a)))
    return h


def grouped_down(h, offsets, experts, D):
    code = weight_dtype_code(h.dtype)
    _need_hip(h, "grouped_down h")
    rows, H = h.shape
    E = len(experts)
    arr = (FfnWeights * E)(*experts)
    y = torch.empty((rows, D), dtype=BF16, device=h.device)
    check(lib.hdmoe_grouped_down(code, ptr(h), ptr(offsets), rows, E, H, D, arr, ptr(y), _stream(h)))
    return y


def ffn_swiglu(x2d, weights, H, weight_dtype):
    """One dense SwiGLU feed-forward as three enqueues. weights: FfnWeights. x2d [rows,D] bf16 -> [rows,D] bf16."""
    _need_hip(x2d, "ffn_swiglu x", BF16)
    rows, D = x2d.shape
    code = weight_dtype_code(weight_dtype)
    nbytes = lib.hdmoe_ffn_workspace_bytes(rows, D, H, code)
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=x2d.device)
    out = torch.empty((rows, D), dtype=BF16, device=x2d.device)
    fw = FfnWeights.from_buffer_copy(weights)
    check(lib.hdmoe_ffn_swiglu(code, ptr(x2d), rows, D, H, ctypes.byref(fw), ptr(out), ptr(ws), ws.numel(),
                               _stream(x2d)))
    return out


def ffn_branch(x2d, weights, H, weight_dtype, scale, shift, gate, tokens_per_batch, eps=1e-6):
    """ln_modulate, ffn_swiglu and gated_residual (x itself) as one call: the same bytes in fewer launches."""
    _need_hip(x2d, "ffn_branch x", BF16)
    rows, D = x2d.shape
    scale, shift, gate = (_per_batch(t, f"ffn_branch {what}", D, x2d.device) for t, what in ((scale, "scale"), (shift, "shift"), (gate, "gate")))
    if tokens_per_batch <= 0 or rows != scale.shape[0] * tokens_per_batch or shift.shape != scale.shape or gate.shape != scale.shape:
        raise ValueError(f"ffn_branch: rows={rows} is not batch={scale.shape[0]} x tokens_per_batch={tokens_per_batch}")
    code = weight_dtype_code(weight_dtype)
    nbytes = lib.hdmoe_ffn_branch_workspace_bytes(rows, D, H, code)
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=x2d.device)
    out = torch.empty((rows, D), dtype=BF16, device=x2d.device)
    fw = FfnWeights.from_buffer_copy(weights)
    check(lib.hdmoe_ffn_branch(code, ptr(x2d), ptr(scale), ptr(shift), ptr(gate), tokens_per_batch, eps, rows, D, H,
                               ctypes.byref(fw), ptr(out), ptr(ws), ws.numel(), _stream(x2d)))
    return out


def layer_layout(T, D, H, Hs, E, code):
    lay = LayerLayout()
    check(lib.hdmoe_layer_layout_get(T, D, H, Hs, E, code, ctypes.byref(lay)))
    return lay


def moe_ffn(x2d, gate_w, experts, shared, H, Hs, weight_dtype, out=None, workspace=None, want_routing=False,
            stage_events=None, modulation=None, tokens_per_batch=None, ln_eps=1e-6, uniform_scale_in=False,
            scale_check=None, fixed_k_cut=False):
    """The whole layer as one enqueue. experts: list of FfnWeights, shared: FfnWeights or None.
    modulation=(shift, scale, gate), each [B, D] bf16, turns the call into the block's feed-forward branch:
    out = x + gate * layer(LayerNorm(x) * (1 + scale) + shift), with T == B * tokens_per_batch.
    uniform_scale_in: accepted and not used (the casting kernel compares the scale_input values on the device and
    casts the tokens once when they agree).
    fixed_k_cut: what is cut along K (the down projection at small token counts; with 16-bit activations the tiles of a last
    round, at any) is taken from the sizes alone instead of from the segment sizes of the call, so that a row's bytes do
    not depend on the routing of the other rows.
    scale_check: optional pinned int32 tensor of one element that the casting kernel sets to 1 when w1 and w3 of a
    feed-forward turn out to cast the tokens differently (the output is then NaN).
    Returns out [T,D] bf16 (and topk_idx int32, topk_weight bf16 when want_routing)."""
    _need_hip(x2d, "moe_ffn x", BF16)
    _need_hip(gate_w, "moe_ffn gate weight", BF16)
    T, D = x2d.shape
    E = len(experts)
    code = weight_dtype_code(weight_dtype)
    nbytes = lib.hdmoe_layer_workspace_bytes(T, D, H, Hs if shared is not None else 0, E, code)
    if nbytes == 0 and T > 0:
        raise _lib.HdmoeError(_lib.lib.hdmoe_layer_layout_get(T, D, H, Hs, E, code, ctypes.byref(LayerLayout())),
                              lib.hdmoe_last_error().decode())
    if workspace is None or workspace.numel() < nbytes:
        workspace = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=x2d.device)
    if out is None:
        out = torch.empty((T, D), dtype=BF16, device=x2d.device)
    args = LayerArgs()
    args.T, args.D, args.H, args.Hs, args.E, args.weight_dtype = T, D, H, (Hs if shared is not None else 0), E, code
    args.x, args.gate_w = ptr(x2d), ptr(gate_w)
    arr = (FfnWeights * E)(*experts)
    args.experts = arr
    sh = None
    if shared is not None:
        sh = FfnWeights.from_buffer_copy(shared)
        args.shared = ctypes.pointer(sh)
    args.out, args.workspace, args.workspace_bytes = ptr(out), ptr(workspace), workspace.numel()
    args.uniform_scale_in = 1 if uniform_scale_in else 0
    args.fixed_k_cut = 1 if fixed_k_cut else 0
    if scale_check is not None:
        if scale_check.dtype != torch.int32 or scale_check.numel() < 1 or not (scale_check.is_cuda or scale_check.is_pinned()):
            raise TypeError("moe_ffn: scale_check must be an int32 tensor on the device or in pinned host memory")
        args.scale_check = ptr(scale_check)
    if modulation is not None:
        shift, scale, gate = (_per_batch(m, "moe_ffn modulation", D, x2d.device) for m in modulation)
        if not tokens_per_batch or T != shift.shape[0] * tokens_per_batch or not (shift.shape == scale.shape == gate.shape):
            raise ValueError(f"moe_ffn: T={T} is not batch={shift.shape[0]} x tokens_per_batch={tokens_per_batch}")
        args.mod_shift, args.mod_scale, args.mod_gate = ptr(shift), ptr(scale), ptr(gate)
        args.tokens_per_batch, args.ln_eps = tokens_per_batch, ln_eps
    idx = tw = None
    if want_routing:
        idx = torch.empty((T, 2), dtype=torch.int32, device=x2d.device)
        tw = torch.empty((T, 2), dtype=BF16, device=x2d.device)
        args.topk_idx, args.topk_weight = ptr(idx), ptr(tw)
    if stage_events is not None:
        # sequence of NUM_STAGES + 1 hipEvent_t handles (ints) created by the caller
        ev = (ctypes.c_void_p * (_lib.NUM_STAGES + 1))(*stage_events)
        args.stage_events = ev
    check(lib.hdmoe_moe_ffn(ctypes.byref(args), _stream(x2d)))
    # the workspace must outlive the enqueued kernels: torch's caching allocator keeps a freed block
    # tied to the stream it was allocated on, so releasing it here is safe for work on that stream
    if want_routing:
        return out, idx, tw
    return out


# ---- e4m3fn with a scale for each block of 128 -------------------------------------------------------------------
# (Calls on a few rows run for about as long as their checks take. _block_calls makes the ordinary ones, with the same checks, and answers
# None where something is to be done first, to be switched or to be refused: that happens here.)

BLOCK = 128
_HERE = contextlib.nullcontext()
_ACT_CODE = {BF16: W_BF16, F16: _lib.W_F16, FP8: W_E4M3FN}
_OUT_CODE = {None: -1, BF16: W_BF16, F16: _lib.W_F16}
if _block_calls is not None:
    _block_calls.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (lib.hdmoe_quant_block_fp8, lib.hdmoe_block_workspace_bytes,
                                                                        lib.hdmoe_block_linear, lib.hdmoe_block_swiglu)))


def _raw_stream(t):
    """_stream without the object around the handle."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _stream_here(t):
    """The current stream's handle where the compiled functions can make the call: they are there, and the tensor is on the current device.
    Else None."""
    if _block_calls is None:
        return None
    d = t.get_device()
    return torch._C._cuda_getCurrentRawStream(d) if d >= 0 and d == torch._C._cuda_getDevice() else None


def _done(r):
    """What a function of _block_calls returned, or the library's error."""
    return check(r) if r.__class__ is int else r


def _on(device):
    """Context in which `device` is the current one."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _blocks(n):
    return -(-n // BLOCK)


def block_scales(rows, K, device):
    """Room for the scales of [rows, K] activations: fp32 [rows, ceil(K / 128)], the scales of one block next to each other."""
    return torch.empty_strided((rows, _blocks(K)), (1, max(rows, 1)), dtype=torch.float32, device=device)


def quant_block_fp8(x):
    """Cast of 16-bit rows with a scale for every 128 values: x [..., K] bf16 or fp16, K a multiple of 16 ->
    (float8_e4m3fn of x's shape, fp32 scales [rows, ceil(K / 128)] as block_scales lays them out).
    scale = max(max|x|, 2^-96) / 448, value = e4m3fn(x * (448 / max(max|x|, 2^-96)))."""
    st = _stream_here(x)
    if st is not None:
        r = _block_calls.cast(x, st)
        if r is not None:
            return _done(r)
    dt = _act_dtype(x, "quant_block_fp8 x")
    _need_hip(x, "quant_block_fp8 x")
    K = x.shape[-1]
    rows = x.numel() // K if K > 0 else 0
    dev = x.device
    with _on(dev):
        q = torch.empty_like(x, dtype=FP8)
        s = block_scales(rows, K, dev)
        check(lib.hdmoe_quant_block_fp8(_ACT_CODE[dt], x.data_ptr(), rows, K, q.data_ptr(), s.data_ptr(), rows, _raw_stream(x)))
    return q, s


def _block_rows(a, scale_a, what):
    """Checks [rows, K] activations, 16-bit or e4m3fn with scales; the scales laid out as block_scales has them (or None)."""
    if a.dim() != 2:
        raise ValueError(f"{what}: expected [rows, K] activations, got {tuple(a.shape)}")
    if a.dtype != FP8:
        _act_dtype(a, what)
        if scale_a is not None:
            raise TypeError(f"{what}: scales belong to float8_e4m3fn activations, got {a.dtype}")
        _need_hip(a, what)
        return None
    _need_hip(a, what)
    if scale_a is None:
        raise TypeError(f"{what}: float8_e4m3fn activations need their scales")
    rows, K = a.shape
    if scale_a.device != a.device or scale_a.dtype != torch.float32 or scale_a.shape != (rows, _blocks(K)):
        raise ValueError(f"{what}: scales must be float32 [{rows}, {_blocks(K)}] on {a.device}, got {scale_a.dtype} "
                         f"{tuple(scale_a.shape)} on {scale_a.device}")
    if not scale_a.t().is_contiguous():
        scale_a = scale_a.t().contiguous().t()
    return scale_a


def _block_matrix(weight, scale, K, index, what, shapes=None):
    """Checks a weight [N, K] and its scales [ceil(N / 128), ceil(K / 128)] on device `index`; shapes: what they have to be (that of the
    experts before), else formed from the weight's. Returns the shapes."""
    if shapes is None:
        N = weight.shape[0] if weight.dim() == 2 else -1
        shapes = ((N, K), (-(-N // BLOCK), -(-K // BLOCK)))
    if weight.dtype is not FP8 or weight.shape != shapes[0] or weight.get_device() != index or not weight.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous float8_e4m3fn weight {list(shapes[0])} on device {index}, got {weight.dtype} "
                         f"{tuple(weight.shape)} on {weight.device}")
    if scale.dtype is not torch.float32 or scale.shape != shapes[1] or scale.get_device() != index or not scale.is_contiguous():
        raise ValueError(f"{what}: expected contiguous float32 scales {list(shapes[1])} on device {index}, got {scale.dtype} "
                         f"{tuple(scale.shape)} on {scale.device}")
    return shapes


def _block_weights(w, entry, K, dtype, index, what, shapes=None):
    """Fills a BlockWeights from (weight, scale, bias or None) or, for gate/up (dtype None), (w1, scale1, w3, scale3)."""
    if dtype is None:
        w1, s1, w3, s3 = entry
        shapes = _block_matrix(w1, s1, K, index, what, shapes)
        _block_matrix(w3, s3, K, index, what, shapes)
        w.weight3, w.scale3 = w3.data_ptr(), s3.data_ptr()
    else:
        w1, s1, bias = entry
        shapes = _block_matrix(w1, s1, K, index, what, shapes)
        if bias is not None:
            if bias.dtype is not dtype or bias.shape != (shapes[0][0],) or bias.get_device() != index or not bias.is_contiguous():
                raise ValueError(f"{what}: expected a contiguous {dtype} bias [{shapes[0][0]}] on device {index}, got {bias.dtype} "
                                 f"{tuple(bias.shape)} on {bias.device}")
            w.bias = bias.data_ptr()
    w.weight, w.scale = w1.data_ptr(), s1.data_ptr()
    return shapes


def _block_out_dtype(a, out_dtype, what):
    if out_dtype is None:
        out_dtype = BF16 if a.dtype == FP8 else a.dtype
    if out_dtype not in ACT_DTYPES or (a.dtype != FP8 and a.dtype != out_dtype):
        raise TypeError(f"{what}: out_dtype must be bfloat16 or float16, and that of 16-bit activations, got {out_dtype}")
    return out_dtype


def _block_experts(a, offsets, experts, perm, dtype, what):
    """(array of BlockWeights, rows of the segments, N); checks offsets and perm."""
    E = len(experts)
    T, K = a.shape
    dev = a.device
    if not 1 <= E <= _lib.BLOCK_MAX_EXPERTS:
        raise ValueError(f"{what}: {E} experts (1 to {_lib.BLOCK_MAX_EXPERTS})")
    if offsets.dtype != torch.int32 or offsets.shape != (E + 1,) or offsets.device != dev or not offsets.is_contiguous():
        raise ValueError(f"{what}: offsets must be contiguous int32 [{E + 1}] on {dev}")
    rows = T
    if perm is not None:
        rows = T * _lib.TOPK
        if perm.dtype != torch.int32 or perm.shape != (rows,) or perm.device != dev or not perm.is_contiguous():
            raise ValueError(f"{what}: perm must be contiguous int32 [{rows}] on {dev}")
    arr = (_lib.BlockWeights * E)()
    shapes, index = None, a.get_device()
    for w, entry in zip(arr, experts):
        shapes = _block_weights(w, entry, K, dtype, index, what, shapes)
    return arr, rows, shapes[0][0]


def _block_call(fn, swiglu, args, a):
    """fn(args) with the working memory that it asks for."""
    if args.rows == 0 and args.rows_static == 0:
        return
    ref = ctypes.byref(args)
    if swiglu or a.dtype is not FP8:
        nbytes = lib.hdmoe_block_workspace_bytes(ref, swiglu)
        if nbytes > 0:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=a.device)
            args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    check(fn(ref, _raw_stream(a)))


def linear_block_fp8(x, weight, scale_weight, bias=None, scale_x=None, out_dtype=None, fixed_k_cut=False):
    """x [rows, K] times weight [N, K]^T (+ bias [N]): weight float8_e4m3fn with fp32 scales scale_weight
    [ceil(N / 128), ceil(K / 128)]; x bf16 or fp16 (cast as quant_block_fp8 does), or float8_e4m3fn with its scales scale_x
    [rows, ceil(K / 128)] (laid out anew unless they are as quant_block_fp8 returns them). -> [rows, N] of x's type (out_dtype, bf16
    unless given, for float8_e4m3fn x). K and N are multiples of 16; x, weight and bias are contiguous and
    start on 16 bytes. The sums are fp32; bias joins them before the one rounding.
    fixed_k_cut: the sums go in one order whatever the number of rows: a row's bytes do not depend on which rows come with it (few rows are
    otherwise dealt along K, up to three times as fast)."""
    st = _stream_here(x)
    if st is not None:
        r = _block_calls.linear(x, weight, scale_weight, bias, scale_x, _OUT_CODE.get(out_dtype, -2), fixed_k_cut, st)
        if r is not None:
            return _done(r)
    what = "linear_block_fp8"
    dt = _block_out_dtype(x, out_dtype, what)
    s = _block_rows(x, scale_x, what + " x")
    rows, K = x.shape
    dev = x.device
    w = _lib.BlockWeights()
    N = _block_weights(w, (weight, scale_weight, bias), K, dt, x.get_device(), what)[0][0]
    with _on(dev):
        out = torch.empty((rows, N), dtype=dt, device=dev)
        if rows > 0:
            args = _lib.BlockArgs()
            args.a_dtype, args.out_dtype = _ACT_CODE[x.dtype], _ACT_CODE[dt]
            args.fixed_k_cut = 1 if fixed_k_cut else 0
            args.rows_static, args.K_static, args.N_static = rows, K, N
            args.shared = ctypes.pointer(w)
            fixed = args.fixed
            fixed.a, fixed.scale_a, fixed.scale_a_stride, fixed.out = x.data_ptr(), ptr(s), rows, out.data_ptr()
            _block_call(lib.hdmoe_block_linear, 0, args, x)
    return out


def grouped_linear_block_fp8(a, offsets, experts, scale_a=None, out_dtype=None, perm=None, shared=None, a_static=None,
                             scale_static=None, fixed_k_cut=False):
    """linear_block_fp8 of every expert over its row segment [offsets[e], offsets[e + 1]) of a [rows, K]. experts: list of
    (weight [N, K], scale, bias [N] or None), at most 32; offsets: int32 [E + 1] on the device, ascending. a as in linear_block_fp8.
    perm: the dispatch's permutation, sorted row r being row perm[r] // 2 of a [T, K]; the output then has 2T rows. Rows that no
    segment holds are not written. -> out [rows, N].
    shared: one more (weight, scale, bias) over all rows of a_static (with scale_static), of sizes of its own, in the same launch;
    -> (out, out_static). fixed_k_cut: see linear_block_fp8."""
    what = "grouped_linear_block_fp8"
    if shared is not None and a.dtype != FP8:
        out_dtype = _block_out_dtype(a, out_dtype, what)
        _block_rows(a, scale_a, what + " a")
        same = a_static is a and scale_static is None
        a, scale_a = quant_block_fp8(a)
        if same:
            a_static, scale_static = a, scale_a
    if shared is not None:
        if a_static is None or a_static.device != a.device:
            raise ValueError(f"{what}: shared needs a_static on {a.device}")
        if a_static.dtype is not FP8 and scale_static is None:
            _block_out_dtype(a_static, _block_out_dtype(a, out_dtype, what), what + " a_static")
            a_static, scale_static = quant_block_fp8(a_static)
    st = _stream_here(a)
    if st is not None:
        r = _block_calls.grouped_linear(a, offsets, experts, scale_a, _OUT_CODE.get(out_dtype, -2), perm, shared, a_static, scale_static, fixed_k_cut, st)
        if r is not None:
            return _done(r)
    dt = _block_out_dtype(a, out_dtype, what)
    sa = _block_rows(a, scale_a, what + " a")
    dev = a.device
    arr, rows, N = _block_experts(a, offsets, experts, perm, dt, what)
    T, K = a.shape
    with _on(dev):
        args = _lib.BlockArgs()
        args.a_dtype, args.out_dtype = _ACT_CODE[a.dtype], _ACT_CODE[dt]
        args.fixed_k_cut = 1 if fixed_k_cut else 0
        out = torch.empty((rows, N), dtype=dt, device=dev)
        if rows > 0:
            args.E, args.rows, args.K, args.N = len(experts), rows, K, N
            if perm is not None:
                args.perm, args.T = perm.data_ptr(), T
            args.offsets = offsets.data_ptr()
            args.experts = arr
            r = args.routed
            r.a, r.scale_a, r.scale_a_stride, r.out = a.data_ptr(), ptr(sa), T, out.data_ptr()
        out_static = None
        if shared is not None:
            s = _block_rows(a_static, scale_static, what + " a_static")
            n, Ks = a_static.shape
            w = _lib.BlockWeights()
            Ns = _block_weights(w, shared, Ks, dt, a.get_device(), what + " shared")[0][0]
            out_static = torch.empty((n, Ns), dtype=dt, device=dev)
            if n > 0:
                args.rows_static, args.K_static, args.N_static = n, Ks, Ns
                args.shared = ctypes.pointer(w)
                f = args.fixed
                f.a, f.scale_a, f.scale_a_stride, f.out = a_static.data_ptr(), s.data_ptr(), n, out_static.data_ptr()
        _block_call(lib.hdmoe_block_linear, 0, args, a)
    return out if shared is None else (out, out_static)


def grouped_swiglu_block_fp8(a, offsets, experts, scale_a=None, perm=None, shared=None, fixed_k_cut=False, exact=False):
    """First half of every expert's SwiGLU feed-forward, silu(a w1^T) * (a w3^T), cast as quant_block_fp8 does:
    experts: list of (w1 [H, K], scale1, w3 [H, K], scale3); a, scale_a, offsets, perm as in grouped_linear_block_fp8.
    -> (h float8_e4m3fn [rows, H], its scales [rows, ceil(H / 128)]); everything before the cast is fp32. Its products are
    exact with `exact`, for fp16 a (not yet cast), and where neither group has more than 64 rows (unless fixed_k_cut); elsewhere the matrix
    cores cut them, which moves 0.23 % of the cast values by a step. exact costs 15 % on few rows, at most 2.4 times on many.
    shared: one more (w1, scale1, w3, scale3) over all rows of a, with a width of its own, in the same launch (with perm);
    -> (h, scales, h_shared, scales_shared). fixed_k_cut: see linear_block_fp8; the products are then the same kind on any number of rows as
    well."""
    st = _stream_here(a)
    if st is not None:
        r = _block_calls.grouped_swiglu(a, offsets, experts, scale_a, perm, shared, fixed_k_cut, exact, st)
        if r is not None:
            return _done(r)
    what = "grouped_swiglu_block_fp8"
    sa = _block_rows(a, scale_a, what + " a")
    dev = a.device
    arr, rows, H = _block_experts(a, offsets, experts, perm, None, what)
    T, K = a.shape
    with _on(dev):
        args = _lib.BlockArgs()
        args.a_dtype, args.out_dtype = _ACT_CODE[a.dtype], W_BF16
        args.fixed_k_cut, args.exact = 1 if fixed_k_cut else 0, 1 if exact else 0
        h = torch.empty((rows, H), dtype=FP8, device=dev)
        sh = block_scales(rows, H, dev)
        if rows > 0:
            args.E, args.rows, args.K, args.N = len(experts), rows, K, H
            if perm is not None:
                args.perm, args.T = perm.data_ptr(), T
            args.offsets = offsets.data_ptr()
            args.experts = arr
            r = args.routed
            r.a, r.scale_a, r.scale_a_stride, r.out = a.data_ptr(), ptr(sa), T, h.data_ptr()
            r.scale_out, r.scale_out_stride = sh.data_ptr(), rows
        if shared is not None:
            w = _lib.BlockWeights()
            Hs = _block_weights(w, shared, K, None, a.get_device(), what + " shared")[0][0]
            h_shared = torch.empty((T, Hs), dtype=FP8, device=dev)
            sh_shared = block_scales(T, Hs, dev)
            if T > 0:
                args.rows_static, args.K_static, args.N_static = T, K, Hs
                args.shared = ctypes.pointer(w)
                f = args.fixed
                f.a, f.scale_a, f.scale_a_stride, f.out = a.data_ptr(), ptr(sa), T, h_shared.data_ptr()
                f.scale_out, f.scale_out_stride = sh_shared.data_ptr(), T
        _block_call(lib.hdmoe_block_swiglu, 1, args, a)
    return (h, sh) if shared is None else (h, sh, h_shared, sh_shared)


def swiglu_block_fp8(x, w1, scale_w1, w3, scale_w3, scale_x=None, fixed_k_cut=False, exact=False):
    """First half of one dense SwiGLU feed-forward, silu(x w1^T) * (x w3^T), cast as quant_block_fp8 does: x and scale_x as in
    linear_block_fp8, fixed_k_cut and exact as in grouped_swiglu_block_fp8 -> (h float8_e4m3fn [rows, H], its scales
    [rows, ceil(H / 128)]), what linear_block_fp8 takes for w2."""
    st = _stream_here(x)
    if st is not None:
        r = _block_calls.swiglu(x, w1, scale_w1, w3, scale_w3, scale_x, fixed_k_cut, exact, st)
        if r is not None:
            return _done(r)
    what = "swiglu_block_fp8"
    s = _block_rows(x, scale_x, what + " x")
    rows, K = x.shape
    dev = x.device
    w = _lib.BlockWeights()
    H = _block_weights(w, (w1, scale_w1, w3, scale_w3), K, None, x.get_device(), what)[0][0]
    with _on(dev):
        h = torch.empty((rows, H), dtype=FP8, device=dev)
        sh = block_scales(rows, H, dev)
        if rows > 0:
            args = _lib.BlockArgs()
            args.a_dtype, args.out_dtype = _ACT_CODE[x.dtype], W_BF16
            args.fixed_k_cut, args.exact = 1 if fixed_k_cut else 0, 1 if exact else 0
            args.rows_static, args.K_static, args.N_static = rows, K, H
            args.shared = ctypes.pointer(w)
            f = args.fixed
            f.a, f.scale_a, f.scale_a_stride, f.out = x.data_ptr(), ptr(s), rows, h.data_ptr()
            f.scale_out, f.scale_out_stride = sh.data_ptr(), rows
            _block_call(lib.hdmoe_block_swiglu, 1, args, x)
    return h, sh


# ---- layer norm and its gradients --------------------------------------------------------------------------------

_T_CODE = {BF16: _lib.T_BF16, F16: _lib.T_F16, torch.float32: _lib.T_F32}
if _row_calls is not None:
    _row_calls.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.hdmoe_layer_norm, lib.hdmoe_layer_norm_backward_workspace_bytes, lib.hdmoe_layer_norm_backward, lib.hdmoe_gate_balance_workspace_bytes,
        lib.hdmoe_gate_balance, lib.hdmoe_gate_balance_backward, lib.hdmoe_adapters_workspace_bytes, lib.hdmoe_add_adapters, lib.hdmoe_add_adapters_backward)))


def _row_call(name, x, *args):
    """The compiled call of that name on `args` and x's current stream, or None: it is not there, x is on another device than the current one, or it
    leaves this call to Python."""
    if _row_calls is None:
        return None
    d = x.get_device()
    if d < 0 or d != torch._C._cuda_getDevice():
        return None
    return _done(getattr(_row_calls, name)(*args, torch._C._cuda_getCurrentRawStream(d)))


def _norm_rows(x, what):
    """(dtype, rows, D) of contiguous rows of bf16, fp16 or fp32 on the device."""
    if x.dtype not in _T_CODE:
        raise TypeError(f"{what}: expected bfloat16, float16 or float32, got {x.dtype}")
    _need_hip(x, what)
    D = x.shape[-1] if x.dim() > 0 else 0
    if not 1 <= D <= _lib.NORM_MAX_D:
        raise ValueError(f"{what}: rows of {D} values (1 to {_lib.NORM_MAX_D})")
    return x.dtype, x.numel() // D, D


def _norm_gain(t, x, shape, what):
    """Code of a gain's type: that of x or fp32."""
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise TypeError(f"{what}: expected {x.dtype} or float32, got {t.dtype}")
    if t.device != x.device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: expected contiguous {list(shape)} on {x.device}, got {tuple(t.shape)} on {t.device}")
    return _T_CODE[t.dtype]


def _norm_gains(x, weight, bias, D, what):
    code = _T_CODE[x.dtype]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            code = _norm_gain(t, x, (D,), f"{what} {name}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"{what}: weight {weight.dtype} and bias {bias.dtype} differ in type")
    return code


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """torch.nn.functional.layer_norm over the last axis: (x - mean) / sqrt(var + eps) * weight + bias. x [..., D] bf16, fp16 or fp32,
    contiguous, D from 1 to 16384; weight, bias [D] of x's type or fp32 (both the same). Statistics are fp32, of the values' differences from
    their mean; the result is rounded once. ln_modulate, with a scale and a shift of each batch item, rounds between its steps."""
    r = _row_call("layer_norm", x, x, weight, bias, eps)
    if r is not None:
        return r
    what = "layer_norm"
    _, rows, D = _norm_rows(x, what + " x")
    code = _norm_gains(x, weight, bias, D, what)
    with _on(x.device):
        out = torch.empty_like(x)
        check(lib.hdmoe_layer_norm(_T_CODE[x.dtype], ptr(x), rows, D, code, ptr(weight), ptr(bias), eps, ptr(out), _raw_stream(x)))
    return out


def _norm_backward(dy, x, weight, dweight, dbias, gain_code, D, rows, per_group, one_plus, eps):
    dx = torch.empty_like(x)
    args = _lib.NormGradArgs()
    args.dtype, args.gain_dtype, args.D, args.one_plus = _T_CODE[x.dtype], gain_code, D, one_plus
    args.rows, args.rows_per_group, args.eps = rows, per_group, eps
    args.dy, args.x, args.weight = ptr(dy), ptr(x), ptr(weight)
    args.dx, args.dweight, args.dbias = ptr(dx), ptr(dweight), ptr(dbias)
    if dweight is not None or dbias is not None:
        nbytes = lib.hdmoe_layer_norm_backward_workspace_bytes(rows, D, per_group)
        if nbytes > 0:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    check(lib.hdmoe_layer_norm_backward(ctypes.byref(args), _raw_stream(x)))
    return dx


def _norm_dy(dy, x, what):
    if dy.dtype != x.dtype or dy.shape != x.shape or dy.device != x.device or not dy.is_contiguous():
        raise ValueError(f"{what}: dy must be contiguous {x.dtype} {list(x.shape)} on {x.device}, got {dy.dtype} {tuple(dy.shape)} on {dy.device}")


def layer_norm_backward(dy, x, weight=None, bias=None, eps=1e-5, gains=True):
    """Gradients of layer_norm(x, weight, bias, eps) from dy, that of its result: (dx, dweight, dbias), None for a weight or bias that is
    None; without `gains` dx alone. Nothing is kept from the forward pass: mean and variance are taken from x again, which is read anyway. dweight and
    dbias are summed over the rows in fp32, in an order that depends on the sizes alone, and have their gains' type."""
    r = _row_call("layer_norm_backward", x, dy, x, weight, bias, eps, gains)
    if r is not None:
        return r
    what = "layer_norm_backward"
    _, rows, D = _norm_rows(x, what + " x")
    _norm_dy(dy, x, what)
    code = _norm_gains(x, weight, bias, D, what)
    with _on(x.device):
        dweight = None if weight is None or not gains else torch.empty_like(weight)
        dbias = None if bias is None or not gains else torch.empty_like(bias)
        dx = _norm_backward(dy, x, weight, dweight, dbias, code, D, rows, rows, 0, eps)
    return dx, dweight, dbias


def ln_modulate_backward(dy, x2d, scale, tokens_per_batch, eps=1e-6):
    """Gradients of LayerNorm(x) * (1 + scale) + shift with one row of scale and shift for tokens_per_batch rows, from dy:
    (dx [T, D], dscale [B, D], dshift [B, D]). bf16 as ln_modulate, whose roundings between its steps count as none here, fp16 or
    fp32. Sums over a batch item's rows are fp32."""
    r = _row_call("ln_modulate_backward", x2d, dy, x2d, scale, tokens_per_batch, eps)
    if r is not None:
        return r
    what = "ln_modulate_backward"
    dt, T, D = _norm_rows(x2d, what + " x")
    if x2d.dim() != 2:
        raise ValueError(f"{what}: expected x [T, D], got {tuple(x2d.shape)}")
    _norm_dy(dy, x2d, what)
    if scale.dim() == 3 and scale.shape[1] == 1:
        scale = scale[:, 0]
    if scale.dim() != 2 or scale.dtype != dt or scale.shape[1] != D or scale.device != x2d.device or not scale.is_contiguous():
        raise ValueError(f"{what}: scale must be contiguous {dt} [batch, {D}] on {x2d.device}, got {scale.dtype} {tuple(scale.shape)} on {scale.device}")
    if tokens_per_batch <= 0 or T != scale.shape[0] * tokens_per_batch:
        raise ValueError(f"{what}: T={T} is not batch={scale.shape[0]} x tokens_per_batch={tokens_per_batch}")
    with _on(x2d.device):
        dscale, dshift = torch.empty_like(scale), torch.empty_like(scale)
        dx = _norm_backward(dy, x2d, scale, dscale, dshift, _T_CODE[dt], D, T, tokens_per_batch, 1, eps)
    return dx, dscale, dshift


# ---- the router's balance loss -----------------------------------------------------------------------------------

def _fit_int32(what, **sizes):
    """ctypes would cut a size that a C int does not hold."""
    if any(v >= 1 << 31 for v in sizes.values()):
        raise ValueError(f"{what}: {', '.join(f'{k}={v}' for k, v in sizes.items())} (each below 2^31)")


def _balance_args(x2d, gate_w, topk_idx, sequences, mask, alpha, what):
    dt = _act_dtype(x2d, what + " x")
    _need_hip(x2d, what + " x")
    dev = x2d.device
    if x2d.dim() != 2 or gate_w.dim() != 2 or topk_idx.dim() != 2 or gate_w.shape[1] != x2d.shape[1] or topk_idx.shape[0] != x2d.shape[0]:
        raise ValueError(f"{what}: expected x [T, D], gate weight [E, D] and topk_idx [T, k], got {tuple(x2d.shape)}, {tuple(gate_w.shape)} and "
                         f"{tuple(topk_idx.shape)}")
    T, D = x2d.shape
    for name, t, dtype in (("gate weight", gate_w, dt), ("topk_idx", topk_idx, torch.int32), ("mask", mask, torch.bool)):
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"{what}: {name} must be {dtype}, got {t.dtype}")
        if t.device != dev or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous on {dev}")
    if mask is not None and mask.numel() != T:
        raise ValueError(f"{what}: a mask of {mask.numel()} for {T} tokens")
    if sequences < 1 or T % sequences != 0:
        raise ValueError(f"{what}: {T} tokens in {sequences} sequences")
    _fit_int32(what, T=T, D=D, sequences=sequences, E=gate_w.shape[0], k=topk_idx.shape[1])
    args = _lib.BalanceArgs()
    args.dtype, args.T, args.sequences, args.D, args.E, args.k, args.alpha = _T_CODE[dt], T, sequences, D, gate_w.shape[0], topk_idx.shape[1], alpha
    args.x, args.gate_w, args.topk_idx, args.mask = ptr(x2d), ptr(gate_w), ptr(topk_idx), ptr(mask)
    return args


def _balance_call(fn, args, x, backward):
    nbytes = lib.hdmoe_gate_balance_workspace_bytes(ctypes.byref(args), backward)
    if nbytes > 0:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    check(fn(ctypes.byref(args), _raw_stream(x)))


def gate_balance(x2d, gate_w, topk_idx, alpha=0.01, sequences=1, mask=None):
    """The router's auxiliary loss for x2d [T, D] (bf16 or fp16, D a multiple of 8), gate_w [E, D] (E up to 16) and the experts that gate_top2 (or any
    other rule) chose, topk_idx int32 [T, k]: (loss, counts, scores) with scores = softmax(x W^T) fp32 [T, E], counts int32 [sequences, E] of the choices
    in each sequence of T / sequences tokens (1: the whole batch, the reference's seq_aux off), and
    loss = alpha * mean over sequences of sum_e (E counts / (k n)) * (mean score of e), an fp32 scalar. mask: bool, T values in any shape; tokens with
    False are left out of counts, means and n, a sequence of nothing else out of the mean. Logits are fp32: gate_top2 rounds them to
    the activations' type before it chooses. Choices outside 0 .. E - 1 are not counted."""
    r = _row_call("gate_balance", x2d, x2d, gate_w, topk_idx, alpha, sequences, mask)
    if r is not None:
        return r
    what = "gate_balance"
    args = _balance_args(x2d, gate_w, topk_idx, sequences, mask, alpha, what)
    with _on(x2d.device):
        dev = x2d.device
        loss = torch.empty((), dtype=torch.float32, device=dev)
        counts = torch.empty((sequences, args.E), dtype=torch.int32, device=dev)
        scores = torch.empty((args.T, args.E), dtype=torch.float32, device=dev)
        args.loss, args.counts, args.scores = ptr(loss), ptr(counts), ptr(scores)
        _balance_call(lib.hdmoe_gate_balance, args, x2d, 0)
    return loss, counts, scores


def gate_balance_backward(dloss, x2d, gate_w, topk_idx, counts, scores, alpha=0.01, mask=None, dweight=None):
    """Gradients (dx, dgate_w) of gate_balance from dloss, an fp32 scalar on the device, and from dweight [T, k] of x's type, that of the
    chosen scores scores[t, topk_idx[t, j]] (what gate_top2 returns beside the experts), if there is one. counts and scores are those
    that gate_balance returned, which also say how many sequences there were; the other arguments are its own. Sums over tokens are fp32, in an order that
    depends on the sizes alone."""
    r = _row_call("gate_balance_backward", x2d, dloss, x2d, gate_w, topk_idx, counts, scores, alpha, mask, dweight)
    if r is not None:
        return r
    what = "gate_balance_backward"
    args = _balance_args(x2d, gate_w, topk_idx, counts.shape[0] if counts.dim() == 2 else 0, mask, alpha, what)
    dev = x2d.device
    for name, t, dtype, shape in (("dloss", dloss, torch.float32, ()), ("counts", counts, torch.int32, (args.sequences, args.E)),
                                  ("scores", scores, torch.float32, (args.T, args.E)), ("dweight", dweight, x2d.dtype, (args.T, args.k))):
        if t is not None and (t.dtype != dtype or t.shape != shape or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be contiguous {dtype} {list(shape)} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    with _on(dev):
        dx, dw = torch.empty_like(x2d), torch.empty_like(gate_w)
        args.counts, args.scores, args.dloss, args.dweight, args.dx, args.dgate_w = ptr(counts), ptr(scores), ptr(dloss), ptr(dweight), ptr(dx), ptr(dw)
        _balance_call(lib.hdmoe_gate_balance_backward, args, x2d, 1)
    return dx, dw


# ---- low-rank adapters of many requests --------------------------------------------------------------------------

def _adapter_args(x, a, b, scale, index, what):
    """AdapterArgs of x [rows, K] (or [..., K]) with the adapters' tensors, all checked."""
    dt = _act_dtype(x, what + " x")
    _need_hip(x, what + " x")
    dev = x.device
    if a.dim() != 3 or b.dim() != 3 or x.dim() < 2:
        raise ValueError(f"{what}: expected x [..., K], a [n, R, K] and b [n, N, R], got {tuple(x.shape)}, {tuple(a.shape)} and {tuple(b.shape)}")
    n, R, K = a.shape
    N = b.shape[1]
    if x.shape[-1] != K or b.shape[0] != n or b.shape[2] != R:
        raise ValueError(f"{what}: x {tuple(x.shape)}, a {tuple(a.shape)} and b {tuple(b.shape)} do not match")
    for name, t, dtype in (("a", a, dt), ("b", b, dt), ("scale", scale, torch.float32), ("index", index, torch.int32)):
        if t.dtype != dtype:
            raise TypeError(f"{what}: {name} must be {dtype}, got {t.dtype}")
        if t.device != dev or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous on {dev}")
    if scale.shape != (n,):
        raise ValueError(f"{what}: scale must be [{n}], got {tuple(scale.shape)}")
    rows = x.numel() // K if K > 0 else 0
    requests = index.numel()
    if rows > 0 and (requests == 0 or rows % requests != 0):
        raise ValueError(f"{what}: {requests} requests do not divide {rows} rows")
    _fit_int32(what, rows=rows, requests=requests, K=K, N=N, n=n, R=R)
    args = _lib.AdapterArgs()
    args.dtype, args.rows, args.requests, args.K, args.N, args.n, args.R = _T_CODE[dt], rows, requests, K, N, n, R
    args.x, args.a, args.b, args.scale, args.index = ptr(x), ptr(a), ptr(b), ptr(scale), ptr(index)
    return args


def _adapter_rows(t, x, N, what):
    if t.dtype != x.dtype or t.shape != (*x.shape[:-1], N) or t.device != x.device or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {x.dtype} {[*x.shape[:-1], N]} on {x.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _adapter_call(fn, args, x, backward):
    nbytes = lib.hdmoe_adapters_workspace_bytes(ctypes.byref(args), backward)
    if nbytes > 0:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    check(fn(ctypes.byref(args), _raw_stream(x)))


def add_adapters(base, x, a, b, scale, index, out=None, fixed_k_cut=False):
    """base + scale[i] * b[i] @ (a[i] @ x) for every row, i the index of the row's request: low-rank adapters of many requests beside one
    Linear, whose result base [..., N] is on x [..., K]. a [n, R, K] and b [n, N, R] of x's type (bf16 or fp16), R up to 256, adapters of a
    smaller rank filled up with zeros; scale [n] fp32. index: int32, one for each request, each of as many rows of x in turn (x [B, S, K] with index [B]; an
    index for each row: index [rows]); negative or from n on: no adapter, and the row is base's. Sums are fp32, the narrow product between the two
    keeps 16 significant bits, the result is rounded once; infinities in a row's own values or adapter, or in the narrow product, can come out as NaN. `out`: takes the result, base itself if it is to be
    added in place; it overlaps nothing else. fixed_k_cut: a row's bytes do not depend on the rows, requests and adapters that come with it (a @ x is otherwise
    cut by their number)."""
    r = _row_call("add_adapters", x, base, x, a, b, scale, index, out, fixed_k_cut)
    if r is not None:
        return r
    what = "add_adapters"
    args = _adapter_args(x, a, b, scale, index, what)
    _adapter_rows(base, x, args.N, what + " base")
    if out is not None and out is not base:
        _adapter_rows(out, x, args.N, what + " out")
    with _on(x.device):
        if out is None:
            out = torch.empty_like(base)
        args.base, args.out, args.fixed_k_cut = ptr(base), ptr(out), bool(fixed_k_cut)
        _adapter_call(lib.hdmoe_add_adapters, args, x, 0)
    return out


def add_adapters_backward(dy, x, a, b, scale, index):
    """Gradients of add_adapters from dy, that of its result and of base: (dx, da, db) of the types of x, a and b. dx is the
    adapters' part alone, 0 for rows without one; da and db are sums over each adapter's rows in fp32, in an order that depends on the sizes alone, 0 for an
    adapter without rows."""
    r = _row_call("add_adapters_backward", x, dy, x, a, b, scale, index)
    if r is not None:
        return r
    what = "add_adapters_backward"
    args = _adapter_args(x, a, b, scale, index, what)
    _adapter_rows(dy, x, args.N, what + " dy")
    with _on(x.device):
        dx, da, db = torch.empty_like(x), torch.empty_like(a), torch.empty_like(b)
        args.dy, args.dx, args.da, args.db = ptr(dy), ptr(dx), ptr(da), ptr(db)
        _adapter_call(lib.hdmoe_add_adapters_backward, args, x, 1)
    return dx, da, db
