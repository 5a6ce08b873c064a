"""Operation classes with the attribute and method contract of ComfyUI's comfy.ops,
restricted to what the HiDream MoE feed-forward uses (Linear, LayerNorm), computing on the
MI355X through libhdmoe, and low-rank adapters beside a Linear (Adapters).

Reference (paths under /root/reference/comfy): ops.py:61-95 cast_bias_weight,
:97-100 CastWeightBiasOp, :103-115 disable_weight_init.Linear, :282-284
manual_cast.Linear, :314-358 fp8_linear, :360-377 fp8_ops, :379-428 scaled_fp8_ops,
:449-473 pick_operations; model_management.py:1055-1072 cast_to, :1353-1375
supports_fp8_compute.

What ModelPatcher relies on and is therefore kept (model_patcher.py:98-107,
151-173, 594-619, 657-722): nn.Linear parameter names (`weight`, `bias`), the class
attributes `comfy_cast_weights`, `weight_function`, `bias_function`, the optional
`scale_weight` / `scale_input` Parameters, and the by-name hooks `convert_weight` /
`set_weight`. A class from here can be handed to a model constructor as
`operations=` or installed through model_options["custom_operations"].

Every forward needs HIP tensors; a CPU tensor raises (the package has no CPU path).
"""
import contextlib
import logging
import types

import weakref

import torch

from . import functional as HF

FP8 = torch.float8_e4m3fn
BF16 = torch.bfloat16

# Optional side stream for weight transfers (the reference's --async-offload,
# model_management.py:1005-1053). None = transfers ride the current stream.
_offload_streams = {}


def set_offload_stream(device, stream):
    """Install (or with None remove) a side stream used for weight casts to `device`.
    Keep it at the default priority."""
    if stream is None:
        _offload_streams.pop(torch.device(device), None)
    else:
        _offload_streams[torch.device(device)] = stream


def get_offload_stream(device):
    s = _offload_streams.get(torch.device(device)) if device is not None else None
    if s is not None:
        s.wait_stream(torch.cuda.current_stream(device))
    return s


def sync_stream(device, stream):
    if stream is not None:
        torch.cuda.current_stream(device).wait_stream(stream)


def cast_to(weight, dtype=None, device=None, non_blocking=False, copy=False, stream=None):
    """model_management.cast_to: dtype/device move of a weight; returns the tensor itself
    when nothing has to change and no copy was asked for."""
    ctx = stream if stream is not None else contextlib.nullcontext()
    if device is None or weight.device == device:
        if not copy and (dtype is None or weight.dtype == dtype):
            return weight
        with ctx:
            return weight.to(dtype=dtype, copy=copy)
    with ctx:
        r = torch.empty_like(weight, dtype=dtype, device=device)
        r.copy_(weight, non_blocking=non_blocking)
    return r


def cast_bias_weight(s, input=None, dtype=None, device=None, bias_dtype=None):
    """ops.cast_bias_weight: bring `s.weight` / `s.bias` to the input's dtype and device and run
    the registered weight/bias functions (LowVramPatch objects) over the copies."""
    if input is not None:
        if dtype is None:
            dtype = input.dtype
        if bias_dtype is None:
            bias_dtype = dtype
        if device is None:
            device = input.device
    offload_stream = get_offload_stream(device)
    fn_ctx = offload_stream if offload_stream is not None else contextlib.nullcontext()
    non_blocking = device is not None and torch.device(device).type == "cuda"

    bias = None
    if s.bias is not None:
        has_fn = len(getattr(s, "bias_function", ())) > 0
        bias = cast_to(s.bias, bias_dtype, device, non_blocking=non_blocking, copy=has_fn, stream=offload_stream)
        if has_fn:
            with fn_ctx:
                for f in s.bias_function:
                    bias = f(bias)

    has_fn = len(getattr(s, "weight_function", ())) > 0
    weight = cast_to(s.weight, dtype, device, non_blocking=non_blocking, copy=has_fn, stream=offload_stream)
    if has_fn:
        with fn_ctx:
            for f in s.weight_function:
                weight = f(weight)
    sync_stream(device, offload_stream)
    return weight, bias


class CastWeightBiasOp:
    comfy_cast_weights = False
    weight_function = []
    bias_function = []


_scale_cache = {}
_scale_epoch = 0


def invalidate_scale_cache():
    """Forget every cached scale_input value. Called when a Linear of this package loads a state dict or takes a new
    weight, and when a kernel reports that a cached value was stale (take_scale_check). The cache only feeds one host
    decision (do w1 and w3 of a feed-forward share their cast factor, i.e. can the fused kernels run); the kernels
    read every scale from the device and verify that decision there, so a stale entry (`p.data.copy_()` does not bump
    the version counter the cache looks at) gives NaN and a dropped cache, never a wrong number."""
    global _scale_epoch
    _scale_epoch += 1
    _scale_cache.clear()


_scale_check_words = {}


def scale_check_word(device):
    """One pinned int32 per device that the layer's casting kernel sets to 1 when the scale_input values it finds on
    the device contradict what the host asserted from its cached copies (w1 and w3 of a feed-forward must cast the
    tokens alike); that call's output is NaN. Reading it costs no synchronisation: the module looks at it at the
    start of every forward and drops the cache (take_scale_check)."""
    t = _scale_check_words.get(device)
    if t is None:
        t = torch.zeros(1, dtype=torch.int32).pin_memory()
        _scale_check_words[device] = t
    return t


def take_scale_check(device):
    """True once after a kernel has raised the device's check word; the scale cache is dropped with it."""
    t = _scale_check_words.get(device)
    if t is None or int(t[0]) == 0:
        return False
    t.zero_()
    invalidate_scale_cache()
    logging.warning("comfyui_amd: a scale_input changed in place since its value was read; the output of the last "
                    "forward that used it is NaN. Cached scale values dropped.")
    return True


def scale_value(p, use_cache=None):
    """Host value of an fp32 scalar Parameter. A host tensor is read directly (no device involved). A device tensor is
    read once per (parameter object, version, address, cache epoch), so steady-state forwards do not synchronise.
    The entry keeps a weak reference to the tensor it was read from: an id or an address alone can be reused by a
    different tensor after the first one is freed. use_cache: None = only for device tensors."""
    if not (p.is_cuda if use_cache is None else use_cache):
        return float(p.detach().float())
    key = id(p)
    hit = _scale_cache.get(key)
    if hit is not None and hit[0]() is p and hit[1] == p._version and hit[2] == p.data_ptr() and hit[4] == _scale_epoch:
        return hit[3]
    if len(_scale_cache) > 4096:
        _scale_cache.clear()
    v = float(p.detach().float().cpu())
    _scale_cache[key] = (weakref.ref(p), p._version, p.data_ptr(), v, _scale_epoch)
    return v


def _linear_bf16(input, weight, bias, fixed_k_cut=False):
    shape = input.shape
    x2 = input.reshape(-1, shape[-1]).contiguous()
    # a bias is added to the fp32 accumulator before the one rounding to bf16, like F.linear's fused epilogue
    out = HF.linear(x2, weight.contiguous(), bias=None if bias is None else bias.contiguous(), fixed_k_cut=fixed_k_cut)
    return out.reshape(*shape[:-1], weight.shape[0])


def _batch_invariant(module):
    """`module.batch_invariant = True` on a Linear: its contraction, and that of its adapters, is never cut along K by the number of rows, so that a row's
    bytes do not depend on which rows come with it. Not an attribute of the reference classes."""
    return module.__dict__.get("batch_invariant", False)


def _fixed_k_cut(lin):
    return {"fixed_k_cut": True} if _batch_invariant(lin) else {}


def _upcast_ready(lin, input):
    """Whether the stored fp8 weight of `lin` can be multiplied in bf16 as it stands (no cast copy of it is made)."""
    return (lin.weight.dtype == FP8 and lin.weight.device == input.device and input.dtype == BF16
            and len(lin.weight_function) == 0 and HF.linear_upcast_fits(lin.weight.shape[1], lin.weight.shape[0])
            and HF.linear_upcast_aligned(lin.weight, input))


def _linear_upcast(lin, input, scale):
    bias = None
    if lin.bias is not None:
        bias = cast_to(lin.bias, input.dtype, input.device, non_blocking=True, copy=len(lin.bias_function) > 0)
        for f in lin.bias_function:
            bias = f(bias)
        bias = bias.contiguous()
    shape = input.shape
    out = HF.linear_upcast(input.reshape(-1, shape[-1]).contiguous(), lin.weight.contiguous(), scale, bias,
                           fixed_k_cut=_batch_invariant(lin))
    return out.reshape(*shape[:-1], lin.weight.shape[0])


class Adapters(torch.nn.Module):
    """Low-rank adapters of many requests beside a Linear of this package: set as `linear.adapters`, they join each result of its forward, after its
    pre-hooks and before its hooks. a [n, R, in], b [n, out, R] in the activations' type, scale [n] fp32 (the usual alpha / rank times the strength),
    whatever the model is cast to. `index`, set before a forward, is int32 on the device with the adapter of each request in the batch (-1: none), each
    request having as many rows as the others. Not in the reference, which patches a LoRA into the weights: these differ between the requests of one
    batch, and the weights stay as they are. One forward of a model at a time: `index` is the module's. Inference only, as the Linear is;
    autograd.add_adapters has the gradients."""

    def __init__(self, a, b, scale):
        super().__init__()
        self.a, self.b = (torch.nn.Parameter(t, requires_grad=False) for t in (a, b))
        self.register_buffer("scale", scale)
        self.index = None
        self._joined = 0       # results so far
        self._rows = None      # an index for each row, while a routed expert is called (functional.dispatch's order)

    def _apply(self, fn, recurse=True):
        """module.to(dtype) moves the scales and leaves their type: they are fp32 beside adapters of any."""
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != scale.dtype:
            self.scale = scale.to(self.scale.device)
        return self

    @classmethod
    def stack(cls, adapters, dtype=None, device=None):
        """Of [(a [r, in], b [out, r], scale)], whose ranks may differ: those below the largest are filled up with zeros."""
        rank = max(a.shape[0] for a, _, _ in adapters)
        pad = torch.nn.functional.pad
        a = torch.stack([pad(a, (0, 0, 0, rank - a.shape[0])) for a, _, _ in adapters])
        b = torch.stack([pad(b, (0, rank - b.shape[1])) for _, b, _ in adapters])
        scale = torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32)
        return cls(a.to(device=device, dtype=dtype).contiguous(), b.to(device=device, dtype=dtype).contiguous(), scale.to(device))

    def forward(self, base, x, fixed_k_cut=False):
        if torch.is_grad_enabled() and (self.a.requires_grad or self.b.requires_grad):
            raise RuntimeError("comfyui_amd.ops.Adapters: a Linear with adapters is inference only; autograd.add_adapters has the gradients")
        index = self.index if self._rows is None else self._rows
        if index is None:
            raise RuntimeError("comfyui_amd.ops.Adapters: set `index`, the adapter of each request, before the forward")
        if x.dim() == 1:      # a row, as the Linear takes it
            return self.forward(base[None], x[None], fixed_k_cut)[0]
        out = HF.add_adapters(base.contiguous(), x.contiguous(), self.a, self.b, self.scale, index, fixed_k_cut=fixed_k_cut)
        self._joined += 1
        return out


def adapters_of(lin):
    """The adapters beside a Linear, or None."""
    return lin.__dict__["_modules"].get("adapters")


class routed_adapters:
    """Context in which the adapters of a module's Linears take T tokens' rows in functional.dispatch's order: row r of the module's input is token
    perm[r] // 2."""

    def __init__(self, module, T, perm):
        self.on = [ad for ad in (adapters_of(l) for l in module.modules() if isinstance(l, torch.nn.Linear)) if isinstance(ad, Adapters)]
        self.T, self.perm = T, perm

    def __enter__(self):
        for ad in self.on:
            if ad.index is None or ad.index.numel() == 0 or self.T % ad.index.numel() != 0:
                raise RuntimeError(f"comfyui_amd.ops.Adapters: `index` must be set and divide the {self.T} tokens of the layer")
        rows = [ad.index.reshape(-1)[self.perm // (HF.TOPK * (self.T // ad.index.numel()))] for ad in self.on]
        for ad, r in zip(self.on, rows):      # all or, where one of them has no such rows, none: __exit__ follows the former alone
            ad._rows = r

    def __exit__(self, *exc):
        for ad in self.on:
            ad._rows = None


class _Forward:
    """The `forward` of a Linear class: of a module it takes the adapters with it, so that pre-hooks have their say about the input of both and hooks see the
    whole result. Of the class (`Linear.forward`) it is the function itself, the product alone."""

    def __init__(self, own):
        def joined(lin, *args, **kwargs):
            if not args and "input" in kwargs:
                args = (kwargs.pop("input"),)
            out = own(lin, *args, **kwargs)
            ad = adapters_of(lin)
            if ad is None or _class_forward(type(lin)) is not self:
                return out      # (a subclass's forward has called its parent's: they join the outer one's result)
            return ad(out, args[0] if args else next(iter(kwargs.values())), **_fixed_k_cut(lin))

        self.own, self.joined = own, joined

    def __get__(self, lin, cls=None):
        return self.own if lin is None else types.MethodType(self.joined, lin)


def _class_forward(cls):
    return next(c.__dict__["forward"] for c in cls.__mro__ if "forward" in c.__dict__)


def call_linear(lin, input):
    """lin(input) of a Linear that may be of another operations class, which knows nothing of Adapters: one that leaves them out is refused."""
    ad = adapters_of(lin)
    if ad is None or isinstance(lin, disable_weight_init.Linear):
        return lin(input)
    return _with_adapters(lin, ad, lin, input)


def _with_adapters(lin, ad, call, *args, **kwargs):
    before = getattr(ad, "_joined", None)
    out = call(*args, **kwargs)
    if before is not None and ad._joined == before:
        raise RuntimeError(f"comfyui_amd.ops.Adapters: beside a {type(lin).__module__}.{type(lin).__qualname__} whose forward leaves them out")
    return out


class disable_weight_init:
    class LayerNorm(torch.nn.LayerNorm, CastWeightBiasOp):
        """Over the last axis, with gradients (autograd.layer_norm) for input, weight and bias."""

        def reset_parameters(self):
            return None

        def _norm(self, input, weight, bias):
            from . import autograd
            if len(self.normalized_shape) != 1:
                raise NotImplementedError("the HIP layer norm is over the last axis")
            if input.shape[-1:] != torch.Size(self.normalized_shape):
                raise ValueError(f"LayerNorm over {tuple(self.normalized_shape)} for an input {tuple(input.shape)}")
            return autograd.layer_norm(input.contiguous(), weight, bias, self.eps)

        def forward_comfy_cast_weights(self, input):
            if self.weight is None:
                return self._norm(input, None, None)
            weight, bias = cast_bias_weight(self, input)
            return self._norm(input, weight, bias)

        def forward(self, *args, **kwargs):
            if self.comfy_cast_weights or len(self.weight_function) > 0 or len(self.bias_function) > 0:
                return self.forward_comfy_cast_weights(*args, **kwargs)
            return self._norm(*args, **kwargs, weight=self.weight, bias=self.bias)

    class Linear(torch.nn.Linear, CastWeightBiasOp):
        def reset_parameters(self):
            return None

        def __init_subclass__(cls, **kwargs):
            super().__init_subclass__(**kwargs)
            own = _class_forward(cls)
            if not isinstance(own, _Forward):
                cls.forward = _Forward(own)

        def __call__(self, *args, **kwargs):
            ad = adapters_of(self)
            if ad is None:
                return super().__call__(*args, **kwargs)
            return _with_adapters(self, ad, super().__call__, *args, **kwargs)     # (a module's or class's `forward` may have been replaced)

        def _load_from_state_dict(self, *args, **kwargs):
            invalidate_scale_cache()   # load_state_dict copies into the Parameters in place
            return super()._load_from_state_dict(*args, **kwargs)

        def forward_comfy_cast_weights(self, input):
            if _upcast_ready(self, input):
                return _linear_upcast(self, input, None)
            weight, bias = cast_bias_weight(self, input)
            return _linear_bf16(input, weight, bias, **_fixed_k_cut(self))

        @_Forward
        def forward(self, *args, **kwargs):
            if self.comfy_cast_weights or len(self.weight_function) > 0 or len(self.bias_function) > 0:
                return self.forward_comfy_cast_weights(*args, **kwargs)
            return _linear_bf16(args[0], self.weight, self.bias, **_fixed_k_cut(self))


class manual_cast(disable_weight_init):
    class Linear(disable_weight_init.Linear):
        comfy_cast_weights = True

    class LayerNorm(disable_weight_init.LayerNorm):
        comfy_cast_weights = True


_ones = {}


def _one(device):
    t = _ones.get(device)
    if t is None:
        t = torch.ones((), dtype=torch.float32, device=device)
        _ones[device] = t
    return t


def fp8_linear(self, input):
    """ops.fp8_linear on the device: quantise the activations to e4m3fn, multiply on the fp8
    matrix cores with fp32 accumulation, scale by scale_input*scale_weight, round to the input
    dtype. Returns None when the weight is not float8_e4m3fn (as the reference does).
    Unlike the reference the caller's input is left untouched when scale_input is None."""
    if self.weight.dtype != FP8:
        return None
    if input.dim() not in (2, 3):
        return None
    if input.dtype != BF16:
        raise TypeError(f"fp8_linear on the HIP path takes bfloat16 activations, got {input.dtype}")
    weight, bias = cast_bias_weight(self, input, dtype=FP8, bias_dtype=input.dtype)
    dev = input.device
    scale_weight = self.scale_weight
    scale_weight = _one(dev) if scale_weight is None else scale_weight.to(dev)
    scale_input = self.scale_input
    if scale_input is not None:
        scale_input = scale_input.to(dev)
    x2 = input.reshape(-1, input.shape[-1]).contiguous()
    xq = HF.quant_fp8(x2, scale_input)
    out = HF.linear(xq, weight.contiguous(), scale_weight, scale_input,
                    bias=None if bias is None else bias.contiguous())
    return out.reshape(*input.shape[:-1], weight.shape[0])


class fp8_ops(manual_cast):
    class Linear(manual_cast.Linear):
        def reset_parameters(self):
            self.scale_weight = None
            self.scale_input = None
            return None

        def forward_comfy_cast_weights(self, input):
            if not self.training:
                # as comfy/ops.py:367-374: whatever goes wrong in the fp8 path is logged and the Linear is
                # computed in the activation dtype instead
                try:
                    out = fp8_linear(self, input)
                    if out is not None:
                        return out
                except Exception as e:
                    logging.info("Exception during fp8 op: {}".format(e))
            weight, bias = cast_bias_weight(self, input)
            return _linear_bf16(input, weight, bias, **_fixed_k_cut(self))


def scaled_fp8_ops(fp8_matrix_mult=False, scale_input=False, override_dtype=None):
    """Class factory mirroring ops.scaled_fp8_ops: Linear weights are stored as `override_dtype`
    (float8_e4m3fn) with an fp32 scalar `scale_weight` and, iff `scale_input`, an fp32 scalar
    `scale_input` (else the attribute is None)."""
    logging.info("Using scaled fp8: fp8 matrix mult: {}, scale input: {}".format(fp8_matrix_mult, scale_input))

    class scaled_fp8_op(manual_cast):
        class Linear(manual_cast.Linear):
            hdmoe_fp8_matrix_mult = fp8_matrix_mult

            def __init__(self, *args, **kwargs):
                if override_dtype is not None:
                    kwargs["dtype"] = override_dtype
                super().__init__(*args, **kwargs)

            def reset_parameters(self):
                if not hasattr(self, "scale_weight"):
                    self.scale_weight = torch.nn.parameter.Parameter(
                        data=torch.ones((), device=self.weight.device, dtype=torch.float32), requires_grad=False)
                if not scale_input:
                    self.scale_input = None
                if not hasattr(self, "scale_input"):
                    self.scale_input = torch.nn.parameter.Parameter(
                        data=torch.ones((), device=self.weight.device, dtype=torch.float32), requires_grad=False)
                return None

            def forward_comfy_cast_weights(self, input):
                if fp8_matrix_mult:
                    out = fp8_linear(self, input)
                    if out is not None:
                        return out
                # no fp8 matmul (ops.py:405-410): the weight is cast to the compute dtype and
                # scale_weight is multiplied onto the smaller of weight and input
                scale = self.scale_weight.to(input.device)
                # resident weights of the usual sizes: multiplied as they are stored, bf16(scale_weight) on the fp32 sum
                # (one rounding where scaling an operand first rounds twice)
                if _upcast_ready(self, input):
                    return _linear_upcast(self, input, scale)
                bias = None
                if (len(self.weight_function) == 0 and self.bias is None and self.weight.dtype == FP8
                        and self.weight.device == input.device):
                    weight = self.weight  # fp8 -> bf16 is exact; the scale kernel reads the fp8 bytes directly
                else:
                    weight, bias = cast_bias_weight(self, input)
                weight = weight.contiguous()
                if weight.numel() < input.numel():
                    return _linear_bf16(input, HF.scale_to_bf16(weight, scale), bias, **_fixed_k_cut(self))
                if weight.dtype == FP8:
                    weight = HF.scale_to_bf16(weight, _one(input.device))
                return _linear_bf16(HF.scale_to_bf16(input.contiguous(), scale), weight, bias, **_fixed_k_cut(self))

            def convert_weight(self, weight, inplace=False, **kwargs):
                s = self.scale_weight.to(device=weight.device, dtype=weight.dtype)
                if inplace:
                    weight *= s
                    return weight
                return weight * s

            def set_weight(self, weight, inplace_update=False, seed=None, return_weight=False, **kwargs):
                from .float_round import stochastic_rounding
                if (weight.is_cuda and self.weight.dtype == torch.float8_e4m3fn and weight.is_contiguous()
                        and weight.dtype in (torch.float32, torch.bfloat16)):
                    # division, float16 rounding and stochastic rounding in one kernel
                    from . import functional as HF
                    scale = self.scale_weight.to(weight.device)
                    own = self.weight.data
                    if (inplace_update and not return_weight and own.device == weight.device and own.shape == weight.shape
                            and own.is_contiguous() and own.data_ptr() % 4 == 0
                            and own.untyped_storage().data_ptr() != weight.untyped_storage().data_ptr()):
                        # straight into the weight: a temporary and its copy would read and write every byte once more
                        HF.stochastic_round_e4m3fn(weight, scale, seed or 0, out=own)
                        return
                    weight = HF.stochastic_round_e4m3fn(weight, scale, seed or 0)
                else:
                    weight = stochastic_rounding(weight / self.scale_weight.to(device=weight.device, dtype=weight.dtype),
                                                 self.weight.dtype, seed=seed)
                if return_weight:
                    return weight
                if inplace_update:
                    self.weight.data.copy_(weight)
                else:
                    self.weight = torch.nn.Parameter(weight, requires_grad=False)

    return scaled_fp8_op


def block_fp8_rows(input):
    """input's rows as the block-scaled operators take them: [rows, K], contiguous, on 16 bytes (a view may start anywhere; it is copied)."""
    x2 = input.reshape(-1, input.shape[-1]).contiguous()
    return x2 if x2.data_ptr() % 16 == 0 else x2.clone()


class block_fp8_ops(manual_cast):
    """Operations class whose Linear weights are float8_e4m3fn with one fp32 scale for every 128 x 128 block
    (`scale_weight` [ceil(out / 128), ceil(in / 128)]) and whose activations are cast with one for every 128 values of a row, as they
    are. bf16 and fp16 activations; in_features and out_features multiples of 16. The reference's scaled-fp8 Linear has one scale for
    a tensor (ops.py:379-428); hooks and attributes are those of that one."""
    class Linear(manual_cast.Linear):
        def __init__(self, *args, **kwargs):
            dtype = kwargs.get("dtype")
            kwargs["dtype"] = FP8
            super().__init__(*args, **kwargs)
            if self.bias is not None:   # stored in the model's type
                self.bias = torch.nn.Parameter(torch.empty(self.out_features, dtype=BF16 if dtype in (None, FP8) else dtype,
                                                           device=self.weight.device))

        def reset_parameters(self):
            if not hasattr(self, "scale_weight"):
                n, k = self.weight.shape
                self.scale_weight = torch.nn.parameter.Parameter(
                    data=torch.ones((HF._blocks(n), HF._blocks(k)), device=self.weight.device, dtype=torch.float32), requires_grad=False)
            return None

        def parts(self, input):
            """(weight, scales, bias) on the input's device, weight functions (LowVramPatch objects) applied to the stored weight."""
            dev = input.device
            if len(self.weight_function) == 0 and len(self.bias_function) == 0 and self.weight.device == dev and self.bias is None:
                weight, bias = self.weight, None
            else:
                weight, bias = cast_bias_weight(self, input, dtype=FP8, bias_dtype=input.dtype)
            return weight.contiguous(), self.scale_weight.to(dev).contiguous(), None if bias is None else bias.contiguous()

        def forward_comfy_cast_weights(self, input):
            weight, scale, bias = self.parts(input)
            return HF.linear_block_fp8(block_fp8_rows(input), weight, scale, bias=bias, fixed_k_cut=_batch_invariant(self)).reshape(*input.shape[:-1], weight.shape[0])

        def _spread(self, weight):
            """scale_weight as one fp32 value per element, on the weight's device (fp16 would lose scales below 2^-25)."""
            s = self.scale_weight.to(device=weight.device, dtype=torch.float32)
            n, k = weight.shape
            return s.repeat_interleave(HF.BLOCK, 0)[:n].repeat_interleave(HF.BLOCK, 1)[:, :k]

        def convert_weight(self, weight, inplace=False, **kwargs):
            s = self._spread(weight)
            if inplace:
                weight *= s
                return weight
            return (weight * s).to(weight.dtype)

        def set_weight(self, weight, inplace_update=False, seed=None, return_weight=False, **kwargs):
            """The stored scales stay: a value past 448 of its block's scale becomes 448 of it, and a block whose scale is 0 stays zero
            whatever a patch adds to it."""
            from .float_round import stochastic_rounding
            s = self._spread(weight)
            weight = torch.where(s != 0, weight / s, torch.zeros_like(s))
            if weight.is_cuda and weight.dtype == torch.float32:
                weight = HF.stochastic_round_e4m3fn(weight.contiguous(), None, seed or 0)
            else:
                weight = stochastic_rounding(weight, FP8, seed=seed)
            if return_weight:
                return weight
            if inplace_update:
                self.weight.data.copy_(weight)
            else:
                self.weight = torch.nn.Parameter(weight, requires_grad=False)


def block_fp8_parts(linears, input):
    """[(weight, scales, bias)] if every one of these is a block_fp8_ops.Linear whose call does nothing more than its class says (no hooks,
    no forward of its own), so that their products can join others' launches; else None."""
    for l in linears:
        if not isinstance(l, block_fp8_ops.Linear):
            return None
        d, cls = l.__dict__, type(l)
        if (d["_forward_hooks"] or d["_forward_pre_hooks"] or "forward" in d or adapters_of(l) is not None or cls.forward is not disable_weight_init.Linear.forward
                or cls.forward_comfy_cast_weights is not block_fp8_ops.Linear.forward_comfy_cast_weights or l.weight.dtype != FP8):
            return None
    return [l.parts(input) for l in linears]


def supports_fp8_compute(device=None):
    """model_management.supports_fp8_compute narrowed to this build's only target: true on a
    gfx950 HIP device (the reference enables fp8 ops for gfx950 with torch >= 2.7 and ROCm >= 6.4,
    model_management.py:351-353)."""
    if not torch.cuda.is_available():
        return False
    try:
        arch = torch.cuda.get_device_properties(device if device is not None else torch.cuda.current_device()).gcnArchName
    except Exception:
        return False
    return "gfx950" in arch


def pick_operations(weight_dtype, compute_dtype, load_device=None, disable_fast_fp8=False, fp8_optimizations=False,
                    scaled_fp8=None, fast_fp8_matrix_mult=False, block_scales=False):
    """ops.pick_operations policy. `fast_fp8_matrix_mult` stands for the reference's
    `--fast fp8_matrix_mult` command-line switch (cli_args.py:142-148), which has no global here. `block_scales`: the
    weights carry a scale for each 128 x 128 block (not in the reference)."""
    if block_scales:
        return block_fp8_ops
    fp8_compute = supports_fp8_compute(load_device)
    if scaled_fp8 is not None:
        return scaled_fp8_ops(fp8_matrix_mult=fp8_compute and fp8_optimizations, scale_input=fp8_optimizations,
                              override_dtype=scaled_fp8)
    if fp8_compute and (fp8_optimizations or fast_fp8_matrix_mult) and not disable_fast_fp8:
        return fp8_ops
    if compute_dtype is None or weight_dtype == compute_dtype:
        return disable_weight_init
    return manual_cast
