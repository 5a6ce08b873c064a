"""The operators of functional.py that have gradients, as functions that torch's autograd goes through: layer norm, the modulated norm in
front of HiDream's feed-forwards, the gate with its balance loss, and adapters beside a Linear. Everything else of this package is inference only.

Each saves its inputs (the norms nothing more, the gate its scores and counts) and calls functional's *_backward. Gradients that arrive strided are made
contiguous first. There is no second derivative.

Captured graphs: torch keeps a gradient accumulator for a leaf for as long as any eager graph of it lives, with the stream of that graph; a backward pass
that is captured meanwhile would make this stream part of the capture and end the process. These functions cannot see whether one lives and refuse
inputs with gradients while a graph is captured, and a captured backward pass of an eager one: there the *_backward functions are called as they are, which
is what they are tested for."""
import torch
from torch.autograd.function import once_differentiable

from . import functional as HF


def _check(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors) and torch.cuda.is_available() \
            and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"autograd.{what}: inputs with gradients while a graph is captured; call functional's {what} and its backward instead")


def _check_backward(what):
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"autograd.{what}: a backward pass while a graph is captured; call functional's {what}_backward instead")


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight, bias)
        ctx.eps = eps
        return HF.layer_norm(x, weight, bias, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_backward("layer_norm")
        x, weight, bias = ctx.saved_tensors
        sums = any(ctx.needs_input_grad[1:3])
        dx, dw, db = HF.layer_norm_backward(dy.contiguous(), x, weight, bias, ctx.eps, gains=sums)
        return dx, dw if ctx.needs_input_grad[1] else None, db if ctx.needs_input_grad[2] else None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """functional.layer_norm with gradients for x, weight and bias."""
    _check("layer_norm", x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, eps)


class _Modulate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2d, scale, shift, tokens_per_batch, eps):
        ctx.save_for_backward(x2d, scale)
        ctx.shapes = scale.shape, shift.shape
        ctx.args = tokens_per_batch, eps
        return HF.ln_modulate(x2d, scale, shift, tokens_per_batch, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_backward("ln_modulate")
        x2d, scale = ctx.saved_tensors
        dx, ds, dsh = HF.ln_modulate_backward(dy.contiguous(), x2d, scale, *ctx.args)
        return dx, ds.view(ctx.shapes[0]), dsh.view(ctx.shapes[1]), None, None


def ln_modulate(x2d, scale, shift, tokens_per_batch, eps=1e-6):
    """functional.ln_modulate with gradients for x2d, scale and shift (its bf16 roundings between steps count as none in them)."""
    _check("ln_modulate", x2d, scale, shift)
    return _Modulate.apply(x2d, scale, shift, tokens_per_batch, eps)


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2d, gate_w, alpha, sequences, mask):
        idx, weight = HF.gate_top2(x2d, gate_w)
        loss, counts, scores = HF.gate_balance(x2d, gate_w, idx, alpha, sequences, mask)
        ctx.save_for_backward(x2d, gate_w, idx, counts, scores, mask)
        ctx.alpha = alpha
        ctx.mark_non_differentiable(idx, counts)
        ctx.set_materialize_grads(False)
        return idx, weight, loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, _, dweight, dloss, __):
        _check_backward("gate_balance")
        x2d, gate_w, idx, counts, scores, mask = ctx.saved_tensors
        if dweight is None and dloss is None:
            return None, None, None, None, None
        if dloss is None:
            dloss = torch.zeros((), dtype=torch.float32, device=x2d.device)
        dx, dw = HF.gate_balance_backward(dloss.contiguous(), x2d, gate_w, idx, counts, scores, ctx.alpha, mask,
                                          None if dweight is None else dweight.contiguous())
        return dx, dw, None, None, None


def gate(x2d, gate_w, alpha=0.01, sequences=1, mask=None):
    """functional.gate_top2 and gate_balance in one: (topk_idx int32 [T, 2], topk_weight [T, 2], loss, counts), with gradients of topk_weight and loss for
    x2d and gate_w. The choice itself has none, and the rounding of logits and scores to the activations' type counts as none. Tokens that the mask takes
    out are routed like the others but have no gradient."""
    _check("gate", x2d, gate_w)
    return _Gate.apply(x2d, gate_w, alpha, sequences, mask)


class _Adapters(torch.autograd.Function):
    @staticmethod
    def forward(ctx, base, x, a, b, scale, index):
        ctx.save_for_backward(x, a, b, scale, index)
        return HF.add_adapters(base, x, a, b, scale, index)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_backward("add_adapters")
        dx = da = db = None
        if any(ctx.needs_input_grad[1:4]):
            dx, da, db = HF.add_adapters_backward(dy.contiguous(), *ctx.saved_tensors)
        need = ctx.needs_input_grad
        return dy if need[0] else None, dx if need[1] else None, da if need[2] else None, db if need[3] else None, None, None


def add_adapters(base, x, a, b, scale, index):
    """functional.add_adapters with gradients for base, x, a and b; that of x is the adapters' part alone (base has its own way back to x, if it has one)."""
    if scale.requires_grad:
        raise RuntimeError("autograd.add_adapters: the scales have no gradient")
    _check("add_adapters", base, x, a, b)
    return _Adapters.apply(base, x, a, b, scale, index)
