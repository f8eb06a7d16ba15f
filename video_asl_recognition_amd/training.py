"""Operators for training the classifier end on frozen features: LayerNorm forward and backward, the classifier's Linear and
softmax cross entropy as one operator, and the global gradient norm with clipping.

    y = layer_norm(x, weight, bias)                                        # autograd
    loss = linear_cross_entropy(x, weight, target, bias)                   # autograd
    loss, dx, dw, db = linear_cross_entropy_grad(x, weight, target, bias)  # both in one call, without autograd
    norm = clip_grads(grads, max_norm)                                     # or clip_grad_norm_(parameters, max_norm)

Every operator is a launch sequence of libaslhip.so on the current stream; torch allocates outputs and workspaces.  Tensors
are fp32 or bf16 on one GPU; sums, statistics, log sum exp and loss are held in fp32 or wider, and results are rounded once.  No
call waits for the GPU.

Two values between are held in fewer bits for bf16 features, except for few rows and a small weight (at most 16 rows, 2^20 weights
and 16384 classes): the softmax's exponentials, as fp16 of 11 significant bits, from which dbias too is added up, and the loss's
gradient with respect to the logits, as bf16, the type that the matrix instructions of the gradient products take.  The latter
is what shows: dx and dweight were measured 0.0019 to 0.0024 (relative 2-norm) off the exact gradient, of which their own rounding
to bf16 is 0.0017.  A caller who wants neither passes fp32 copies of features and weight: everything is then as good as fp32 sums.

The loss alone holds per row and 32 to 128 classes a maximum and a sum, no logits.  With gradients the exponentials are held, for
as many rows at a time as take 4 GiB (2 bytes an entry for bf16 features, 4 for fp32, 10 for large fp32 problems, whose gradient
is held as three bf16 parts as well), or 256 rows.
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


_HERE = nullcontext()


def _on(index: int):
    """kernels are launched on the device their tensors live on, whichever is current"""
    return _HERE if index == torch.cuda.current_device() else torch.cuda.device(index)


def _device(x: torch.Tensor, **tensors) -> int:
    """index of the GPU that all of them are on"""
    index = x.get_device()
    if index < 0:
        raise ValueError(f"tensors must be on the GPU, got {x.device}")
    for name, t in tensors.items():
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, expected {x.device}")
    return index


def _countable(t: torch.Tensor, what: str):
    """the C parameters count rows and columns in 32 bits, and ctypes would cut a larger number without a word"""
    d = t.shape[-1]
    if d >> 31 or (t.numel() >> 31 and t.numel() // d >> 31):
        raise ValueError(f"{what} must be of fewer than 2^31 rows and columns, got {tuple(t.shape)}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., d] -> [rows, d] with unit stride along d and rows that do not overlap; a view where the strides allow it"""
    if t.dim() == 2 and t.is_contiguous():
        return t
    d = t.shape[-1]
    t = t.reshape(-1, d) if d else t.reshape(0, 0)
    if (d > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# handle of a device's current stream; the shortcut saves the stream object that torch.cuda.current_stream builds (1.7 us of a
# small call's 10)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _like(t: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """contiguous, of t's shape; empty_like, where it keeps the strides anyway, is the cheaper call"""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _bytes(n: int, what: str) -> int:
    if n < 0:
        L.check(int(n), what)
    return max(int(n), 16)


# ---------------------------------------------------------------------------------------------- LayerNorm
def _check_norm(x, weight, bias):
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"x must be [..., d] with d >= 1, got {tuple(shape)}")
    _countable(x, "x")
    d = shape[-1]
    if (weight is not None and weight.shape != (d,)) or (bias is not None and bias.shape != (d,)):
        raise ValueError(f"weight and bias must be [{d}], got {[None if t is None else tuple(t.shape) for t in (weight, bias)]}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight is {weight.dtype}, bias {bias.dtype}: one type for both")
    w = weight if weight is not None else bias
    return d, _type(x, "x"), (_type(w, "weight") if w is not None else L.F32)


def layer_norm_fwd(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float = 1e-5,
                   out_dtype: Optional[torch.dtype] = None):
    """x [..., d] -> (y [..., d], mean [...], rstd [...]): LayerNorm over the last dimension, y in `out_dtype` (default: x's),
    and the fp32 statistics that layer_norm_bwd takes."""
    d, xt, wt = _check_norm(x, weight, bias)
    index = _device(x, weight=weight, bias=bias)
    x2 = _rows(x)
    y = _like(x, out_dtype)
    mean, rstd = x.new_empty((2,) + x.shape[:-1], dtype=torch.float32).unbind(0)
    w = weight.contiguous() if weight is not None else None
    b = bias.contiguous() if bias is not None else None
    p = L.LayerNormParams(x2.shape[0], d, _ld(x2), d, d, xt, wt, _type(y, "out_dtype"), eps)
    with _on(index):
        L.check(L.lib.asl_layernorm_fwd(C.byref(p), x2.data_ptr(), _ptr(w), _ptr(b), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                        _stream(index)), "layer_norm_fwd")
    return y, mean, rstd


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor):
    """(dx, dweight, dbias) of layer_norm_fwd: dx in x's type, the other two in the weight's (fp32 without one)."""
    d, xt, wt = _check_norm(x, weight, None)
    index = _device(x, weight=weight, dy=dy, mean=mean, rstd=rstd)
    if dy.shape != x.shape:
        raise ValueError(f"dy is {tuple(dy.shape)}, x {tuple(x.shape)}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.shape != x.shape[:-1]:
            raise ValueError(f"{name} must be float32 {tuple(x.shape[:-1])}, got {t.dtype} {tuple(t.shape)}")
    x2, dy2, mean, rstd = _rows(x), _rows(dy), mean.contiguous(), rstd.contiguous()
    w = weight.contiguous() if weight is not None else None
    dx = _like(x)
    dw = _like(weight) if weight is not None else x.new_empty(d, dtype=torch.float32)
    db = torch.empty_like(dw)
    p = L.LayerNormParams(x2.shape[0], d, _ld(x2), _ld(dy2), d, xt, wt, _type(dy, "dy"), 0.0)
    ws = x.new_empty(_bytes(L.lib.asl_layernorm_bwd_workspace(C.byref(p)), "layer_norm_bwd"), dtype=torch.uint8)
    with _on(index):
        L.check(L.lib.asl_layernorm_bwd(C.byref(p), dy2.data_ptr(), x2.data_ptr(), _ptr(w), mean.data_ptr(), rstd.data_ptr(),
                                        dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), _stream(index)), "layer_norm_bwd")
    return dx, dw, db


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
    _countable(x, "x")
    _countable(weight, "weight")
    index = _device(x, weight=weight, target=target, bias=bias)
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
    return index


def _xent(x, weight, target, bias, ignore_index, label_smoothing, reduction):
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index must be a 64-bit number, got {ignore_index}")
    index = _check_xent(x, weight, target, bias, reduction, label_smoothing)
    x2, w2, t = _rows(x), _rows(weight), target.contiguous()
    b = bias.contiguous() if bias is not None else None
    p = L.XentParams(x2.shape[0], w2.shape[0], w2.shape[1], _type(x, "x"), _type(b, "bias") if b is not None else L.F32,
                     _REDUCTIONS[reduction], _ld(x2), _ld(w2), ignore_index, label_smoothing, 0)
    return index, x2, w2, t, b, p


def linear_cross_entropy_fwd(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                             ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean"):
    """(loss, lse) of cross_entropy(linear(x, weight, bias), target): x [..., d], weight [classes, d] of the same type, target
    int64 [...].  loss is fp32, 0-d or (reduction "none") of target's shape; lse, fp32 of target's shape, is log sum exp of
    the logits."""
    index, x2, w2, t, b, p = _xent(x, weight, target, bias, ignore_index, label_smoothing, reduction)
    loss = x.new_empty(target.shape if reduction == "none" else (), dtype=torch.float32)
    lse = x.new_empty(target.shape, dtype=torch.float32)
    ws = x.new_empty(_bytes(L.lib.asl_linear_xent_workspace(C.byref(p), x2.data_ptr(), w2.data_ptr(), 0), "linear_cross_entropy"),
                     dtype=torch.uint8)
    if loss.numel():
        with _on(index):
            L.check(L.lib.asl_linear_xent_fwd(C.byref(p), x2.data_ptr(), w2.data_ptr(), _ptr(b), t.data_ptr(), loss.data_ptr(),
                                              lse.data_ptr(), ws.data_ptr(), _stream(index)), "linear_cross_entropy_fwd")
    return loss, lse


def _xent_grad(x, weight, target, bias, upstream, ignore_index, label_smoothing, reduction, want):
    index, x2, w2, t, b, p = _xent(x, weight, target, bias, ignore_index, label_smoothing, reduction)
    loss = x.new_empty(target.shape if reduction == "none" else (), dtype=torch.float32)
    dx = _like(x) if want[0] else None
    dw = _like(weight) if want[1] else None
    db = _like(bias) if want[2] and bias is not None else None
    ws = x.new_empty(_bytes(L.lib.asl_linear_xent_workspace(C.byref(p), x2.data_ptr(), w2.data_ptr(), 1), "linear_cross_entropy"),
                     dtype=torch.uint8)
    # a 0-row "none" loss has no storage: the entry point wants an address all the same and writes nothing there
    with _on(index):
        L.check(L.lib.asl_linear_xent_grad(C.byref(p), x2.data_ptr(), w2.data_ptr(), _ptr(b), t.data_ptr(), _ptr(upstream),
                                           loss.data_ptr() or ws.data_ptr(), None, _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(),
                                           _stream(index)), "linear_cross_entropy_grad")
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


def _layout(tensors, index, what):
    """(types, addresses, whether all are contiguous) of tensors that must be dense and on one GPU; a few C-level passes over
    the list, because a model has hundreds of them"""
    n = len(tensors)
    where = list(map(torch.Tensor.get_device, tensors))
    if where.count(index) != n:
        i = next(i for i, w in enumerate(where) if w != index)
        raise ValueError(f"{what} {i} is on {tensors[i].device}, expected cuda:{index}")
    types = [_TYPES.get(t.dtype, -1) for t in tensors]
    if -1 in types:
        i = types.index(-1)
        raise ValueError(f"{what} {i} must be float32 or bfloat16, got {tensors[i].dtype}")
    flat = all(map(torch.Tensor.is_contiguous, tensors))
    if not flat:
        for i, t in enumerate(tensors):
            if not _dense(t):
                raise ValueError(f"{what} {i} is not dense: strides {t.stride()} for {tuple(t.shape)}")
    return array.array("i", types), array.array("Q", list(map(torch.Tensor.data_ptr, tensors))), flat


def _clip(grads: Sequence[torch.Tensor], max_norm, norm_type, out: Optional[Sequence[torch.Tensor]]):
    grads = list(grads)
    if norm_type not in (2, float("inf")):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    if not grads:
        raise ValueError("no gradients")
    index, n = grads[0].get_device(), len(grads)
    if index < 0:
        raise ValueError(f"gradients must be on the GPU, got {grads[0].device}")
    types, ptrs, flat = _layout(grads, index, "gradient")
    numel = array.array("q", list(map(torch.Tensor.numel, grads)))
    otypes = optrs = None
    if out is not None:
        out = list(out)
        otypes, optrs, oflat = _layout(out, index, "output")
        if len(out) != n or list(map(torch.Tensor.numel, out)) != numel.tolist():
            raise ValueError(f"{n} gradients, {len(out)} outputs, or not tensor for tensor the same number of elements")
        if not (flat and oflat):
            for i, (g, o) in enumerate(zip(grads, out)):
                if not (g.is_contiguous() and o.is_contiguous()) and (g.shape != o.shape or g.stride() != o.stride()):
                    raise ValueError(f"output {i} has strides {o.stride()}, gradient {g.stride()}")
    elif max_norm is not None:
        otypes, optrs = types, ptrs
    addr = lambda a: a.buffer_info()[0] if a is not None else None
    norm = grads[0].new_empty((), dtype=torch.float32)
    ws = norm.new_empty(_bytes(L.lib.asl_grad_clip_workspace(n, addr(numel)), "clip_grads"), dtype=torch.uint8)
    with _on(index):
        L.check(L.lib.asl_grad_clip(n, addr(ptrs), addr(numel), addr(types), addr(optrs), addr(otypes),
                                    0.0 if max_norm is None else float(max_norm), int(norm_type != 2), norm.data_ptr(), ws.data_ptr(),
                                    _stream(index)), "clip_grads")
    if otypes is not None:              # written through their addresses: a backward that still needs one of them has to be told
        torch.autograd.graph.increment_version(grads if out is None else out)
    return norm


@torch.no_grad()
def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, norm_type inf, the largest magnitude) over all elements of all tensors: fp32, 0-d, on the GPU."""
    return _clip(grads, None, norm_type, None)


@torch.no_grad()
def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the gradients by min(1, max_norm / (norm + 1e-6)), in place or into `out` (tensor for tensor, fp32 or bf16 each, of
    the same strides or both contiguous: bf16 gradients into an optimizer's fp32 buffers in the same pass), and returns the
    norm they had.  Tensors that are written may not overlap, each other or a gradient that is not their own; autograd sees them as
    written in place.  NaN in, NaN out."""
    return _clip(grads, max_norm, norm_type, out)


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ for norm_type 2 and inf and parameters on one GPU: clips their .grad in place, returns the
    norm."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    parameters = list(parameters)
    grads: List[torch.Tensor] = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=parameters[0].device if parameters else None)
    return _clip(grads, max_norm, norm_type, None)
