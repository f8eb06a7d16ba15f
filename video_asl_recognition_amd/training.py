"""Operators for training the classifier end on frozen features: LayerNorm forward and backward, the classifier's Linear and
softmax cross entropy as one operator that never holds the logits, and the global gradient norm with clipping.

    y = layer_norm(x, weight, bias)                                        # autograd
    loss = linear_cross_entropy(x, weight, target, bias)                   # autograd
    loss, dx, dw, db = linear_cross_entropy_grad(x, weight, target, bias)  # both in one call, without autograd
    norm = clip_grads(grads, max_norm)                                     # or clip_grad_norm_(parameters, max_norm)

Every operator is a launch sequence of libaslhip.so on the current stream; torch allocates outputs and workspaces.  Tensors
are fp32 or bf16 on one GPU; sums, statistics and softmax are held in fp32 or wider, results are rounded once (the loss's
gradient with respect to bf16 logits is additionally rounded to bf16, as the operand of the gradient products).  No call
waits for the GPU.
"""
from __future__ import annotations

import array
import ctypes as C
from contextlib import nullcontext
from typing import Iterable, List, Optional, Sequence, Union

import torch

from . import _lib as L

_TYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16}
_REDUCTIONS = {"none": L.REDUCE_NONE, "sum": L.REDUCE_SUM, "mean": L.REDUCE_MEAN}


def _type(t: torch.Tensor, what: str) -> int:
    c = _TYPES.get(t.dtype)
    if c is None:
        raise ValueError(f"{what} must be float32 or bfloat16, got {t.dtype}")
    return c


def _on(dev: torch.device):
    """kernels are launched on the device their tensors live on, whichever is current"""
    return nullcontext() if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _same_device(dev, **tensors):
    if dev.type != "cuda":
        raise ValueError(f"tensors must be on the GPU, got {dev}")
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., d] -> [rows, d] with unit stride along d and rows that do not overlap; a view where the strides allow it"""
    d = t.shape[-1]
    t = t.reshape(-1, d) if d else t.reshape(0, 0)
    if (d > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def _bytes(n: int, what: str) -> int:
    if n < 0:
        L.check(int(n), what)
    return max(int(n), 16)


# ---------------------------------------------------------------------------------------------- LayerNorm
def _check_norm(x, weight, bias):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., d] with d >= 1, got {tuple(x.shape)}")
    d = x.shape[-1]
    _same_device(x.device, weight=weight, bias=bias)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (d,):
            raise ValueError(f"{name} must be [{d}], got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight is {weight.dtype}, bias {bias.dtype}: one type for both")
    w = weight if weight is not None else bias
    return _type(x, "x"), (_type(w, "weight") if w is not None else L.F32)


def layer_norm_fwd(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float = 1e-5,
                   out_dtype: Optional[torch.dtype] = None):
    """x [..., d] -> (y [..., d], mean [...], rstd [...]): LayerNorm over the last dimension, y in `out_dtype` (default: x's),
    and the fp32 statistics that layer_norm_bwd takes."""
    xt, wt = _check_norm(x, weight, bias)
    dev, lead, d = x.device, x.shape[:-1], x.shape[-1]
    x2 = _rows(x)
    rows = x2.shape[0]
    y = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=dev)
    stats = torch.empty((2,) + tuple(lead), dtype=torch.float32, device=dev)
    mean, rstd = stats[0], stats[1]
    w = weight.contiguous() if weight is not None else None
    b = bias.contiguous() if bias is not None else None
    p = L.LayerNormParams(rows, d, _ld(x2), d, d, xt, wt, _type(y, "out_dtype"), eps)
    with _on(dev):
        L.check(L.lib.asl_layernorm_fwd(C.byref(p), _ptr(x2), _ptr(w), _ptr(b), _ptr(y), _ptr(mean), _ptr(rstd), _stream(dev)),
                "layer_norm_fwd")
    return y, mean, rstd


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor):
    """(dx, dweight, dbias) of layer_norm_fwd: dx in x's type, the other two in the weight's (fp32 without one)."""
    xt, wt = _check_norm(x, weight, None)
    dev, lead, d = x.device, x.shape[:-1], x.shape[-1]
    _same_device(dev, dy=dy, mean=mean, rstd=rstd)
    if dy.shape != x.shape:
        raise ValueError(f"dy is {tuple(dy.shape)}, x {tuple(x.shape)}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.shape != lead:
            raise ValueError(f"{name} must be float32 {tuple(lead)}, got {t.dtype} {tuple(t.shape)}")
    x2, dy2, mean, rstd = _rows(x), _rows(dy), mean.contiguous(), rstd.contiguous()
    w = weight.contiguous() if weight is not None else None
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dwb = torch.empty(2, d, dtype=weight.dtype if weight is not None else torch.float32, device=dev)
    p = L.LayerNormParams(x2.shape[0], d, _ld(x2), _ld(dy2), d, xt, wt, _type(dy, "dy"), 0.0)
    ws = torch.empty(_bytes(L.lib.asl_layernorm_bwd_workspace(C.byref(p)), "layer_norm_bwd"), dtype=torch.uint8, device=dev)
    base = dwb.data_ptr()
    with _on(dev):
        L.check(L.lib.asl_layernorm_bwd(C.byref(p), _ptr(dy2), _ptr(x2), _ptr(w), _ptr(mean), _ptr(rstd), _ptr(dx), base,
                                        base + d * dwb.element_size(), _ptr(ws), _stream(dev)), "layer_norm_bwd")
    return dx, dwb[0], dwb[1]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps, out_dtype)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_bwd(dy, x, weight, mean, rstd)
        return (dx if ctx.needs_input_grad[0] else None, dw if ctx.needs_input_grad[1] else None,
                db.to(ctx.bias_dtype) if ctx.needs_input_grad[2] else None, None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """nn.functional.layer_norm over the last dimension, differentiable (once)."""
    return _LayerNorm.apply(x, weight, bias, eps, out_dtype)


# ---------------------------------------------------------------------------------------------- Linear + cross entropy
def _check_xent(x, weight, target, bias, reduction, label_smoothing):
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or min(weight.shape) < 1:
        raise ValueError(f"x must be [..., d] and weight [classes, d], got {tuple(x.shape)} and {tuple(weight.shape)}")
    _same_device(x.device, weight=weight, target=target, bias=bias)
    if x.dtype != weight.dtype:
        raise ValueError(f"x is {x.dtype}, weight {weight.dtype}: one type for both")
    if target.dtype != torch.int64 or target.shape != x.shape[:-1]:
        raise ValueError(f"target must be int64 {tuple(x.shape[:-1])}, got {target.dtype} {tuple(target.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")


def _xent(x, weight, target, bias, ignore_index, label_smoothing, reduction):
    _check_xent(x, weight, target, bias, reduction, label_smoothing)
    x2, w2, t = _rows(x), _rows(weight), target.contiguous()
    b = bias.contiguous() if bias is not None else None
    p = L.XentParams(x2.shape[0], w2.shape[0], w2.shape[1], _type(x, "x"), _type(b, "bias") if b is not None else L.F32,
                     _REDUCTIONS[reduction], _ld(x2), _ld(w2), ignore_index, label_smoothing, 0)
    return x2, w2, t, b, p


def linear_cross_entropy_fwd(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                             ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean"):
    """(loss, lse) of cross_entropy(linear(x, weight, bias), target): x [..., d], weight [classes, d] of the same type, target
    int64 [...].  loss is fp32, 0-d or (reduction "none") of target's shape; lse, fp32 of target's shape, is log sum exp of
    the logits."""
    x2, w2, t, b, p = _xent(x, weight, target, bias, ignore_index, label_smoothing, reduction)
    dev = x.device
    loss = torch.empty(target.shape if reduction == "none" else (), dtype=torch.float32, device=dev)
    lse = torch.empty(target.shape, dtype=torch.float32, device=dev)
    ws = torch.empty(_bytes(L.lib.asl_linear_xent_workspace(C.byref(p), _ptr(x2), _ptr(w2), 0), "linear_cross_entropy"), dtype=torch.uint8, device=dev)
    if loss.numel():
        with _on(dev):
            L.check(L.lib.asl_linear_xent_fwd(C.byref(p), _ptr(x2), _ptr(w2), _ptr(b), _ptr(t), _ptr(loss), _ptr(lse), _ptr(ws),
                                              _stream(dev)), "linear_cross_entropy_fwd")
    return loss, lse


def _xent_grad(x, weight, target, bias, upstream, ignore_index, label_smoothing, reduction, want):
    x2, w2, t, b, p = _xent(x, weight, target, bias, ignore_index, label_smoothing, reduction)
    dev = x.device
    loss = torch.empty(target.shape if reduction == "none" else (), dtype=torch.float32, device=dev)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want[0] else None
    dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if want[1] else None
    db = torch.empty(bias.shape, dtype=bias.dtype, device=dev) if want[2] and bias is not None else None
    ws = torch.empty(_bytes(L.lib.asl_linear_xent_workspace(C.byref(p), _ptr(x2), _ptr(w2), 1), "linear_cross_entropy"), dtype=torch.uint8, device=dev)
    # a 0-row "none" loss has no storage: the entry point wants an address all the same and writes nothing there
    with _on(dev):
        L.check(L.lib.asl_linear_xent_grad(C.byref(p), _ptr(x2), _ptr(w2), _ptr(b), _ptr(t), _ptr(upstream),
                                           _ptr(loss) or _ptr(ws), None, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), _stream(dev)),
                "linear_cross_entropy_grad")
    return loss, dx, dw, db


def linear_cross_entropy_grad(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                              ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean"):
    """(loss, dx, dweight, dbias) in one call: the loss of linear_cross_entropy_fwd and its gradients (of the sum of the rows'
    losses for reduction "none"); dbias is None without a bias.  A training step that calls this instead of going through
    autograd computes the logits' product once instead of twice."""
    return _xent_grad(x, weight, target, bias, None, ignore_index, label_smoothing, reduction, (True, True, True))


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, bias, ignore_index, label_smoothing, reduction):
        loss, _ = linear_cross_entropy_fwd(x, weight, target, bias, ignore_index=ignore_index, label_smoothing=label_smoothing,
                                           reduction=reduction)
        ctx.save_for_backward(x, weight, target, bias)
        ctx.how = (ignore_index, label_smoothing, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, weight, target, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        _, dx, dw, db = _xent_grad(x, weight, target, bias, g.float().contiguous(), *ctx.how, (need[0], need[1], need[3]))
        return dx, dw, None, db, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                         ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean") -> torch.Tensor:
    """The loss of linear_cross_entropy_fwd, differentiable (once) in x, weight and bias.  Backward forms the logits anew
    rather than keeping them."""
    return _LinearCrossEntropy.apply(x, weight, target, bias, ignore_index, label_smoothing, reduction)


# ---------------------------------------------------------------------------------------------- gradient norm and clipping
def _dense(t: torch.Tensor) -> bool:
    """every element of one block of memory exactly once, in whatever order"""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _clip(grads: Sequence[torch.Tensor], max_norm, norm_type, out: Optional[Sequence[torch.Tensor]], device):
    grads = list(grads)
    norm_type = float(norm_type)
    if norm_type not in (2.0, float("inf")):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    if not grads and device is None:
        raise ValueError("no gradients")
    dev = grads[0].device if grads else torch.device(device)
    if dev.type != "cuda":
        raise ValueError(f"gradients must be on the GPU, got {dev}")
    if out is None and max_norm is not None:
        out = grads
    elif out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"{len(grads)} gradients, {len(out)} outputs")
    kinds, okinds = array.array("i"), array.array("i")
    for i, g in enumerate(grads):
        if g.device != dev:
            raise ValueError(f"gradient {i} is on {g.device}, expected {dev}")
        kinds.append(_type(g, "gradients"))
        if not _dense(g):
            raise ValueError(f"gradient {i} is not dense: strides {g.stride()} for {tuple(g.shape)}")
        if out is not None and out is not grads:
            o = out[i]
            if o.device != dev or o.shape != g.shape:
                raise ValueError(f"output {i} is {tuple(o.shape)} on {o.device}, gradient {tuple(g.shape)} on {dev}")
            if o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous()):
                raise ValueError(f"output {i} has strides {o.stride()}, gradient {g.stride()}")
            okinds.append(_type(o, "outputs"))
    n = len(grads)
    ptrs = array.array("Q", [g.data_ptr() for g in grads])
    numel = array.array("q", [g.numel() for g in grads])
    optrs = ptrs if out is grads else array.array("Q", [o.data_ptr() for o in out]) if out is not None else None
    if out is grads:
        okinds = kinds
    addr = lambda a: a.buffer_info()[0] if a is not None and n else None
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(_bytes(L.lib.asl_grad_clip_workspace(n, addr(numel)), "clip_grads"), dtype=torch.uint8, device=dev)
    with _on(dev):
        L.check(L.lib.asl_grad_clip(n, addr(ptrs), addr(numel), addr(kinds), addr(optrs), addr(okinds) if optrs is not None else None,
                                    0.0 if max_norm is None else float(max_norm), int(norm_type != 2.0), _ptr(norm), _ptr(ws),
                                    _stream(dev)), "clip_grads")
    return norm


@torch.no_grad()
def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, norm_type inf, the largest magnitude) over all elements of all tensors: fp32, 0-d, on the GPU."""
    return _clip(grads, None, norm_type, None, None)


@torch.no_grad()
def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the gradients by min(1, max_norm / (norm + 1e-6)), in place or into `out` (tensor for tensor, fp32 or bf16 each:
    bf16 gradients into an optimizer's fp32 buffers in the same pass), and returns the norm they had.  A tensor may not be
    listed twice.  NaN in, NaN out."""
    return _clip(grads, max_norm, norm_type, out, None)


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ for norm_type 2 and inf: clips the parameters' .grad in place, returns their norm."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    parameters = list(parameters)
    grads: List[torch.Tensor] = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=parameters[0].device if parameters else None)
    return _clip(grads, max_norm, norm_type, None, None)
