"""Training operators on PyTorch-ROCm tensors, reached as `tilec.ext.*`: layer
norm and root mean square norm with their gradients, the cross entropy of a
linear layer's outputs and its gradients, the norm of a model's gradients with
clipping, and an AdamW step over many tensors.

They are what a training step needs beside the products (`matrix_mul`) and the
sums (`sum`) of its linear layers, and follow the same rules: arguments are
checked before anything is enqueued (ValueError for shapes, TypeError for
types and devices), work goes to the current stream of the tensors' device,
and nothing synchronises.  Scratch that carries values from one kernel of a call
to the next is torch's allocator's, each call's own: calls of other host threads
on the same stream may put their kernels in between.
Like those two they are plain functions with no autograd of their own.
"""

import ctypes
from functools import lru_cache

import torch

from . import _lib
from .ext import _current_device, _raw_stream, _stream_captured, _tuned, counters_for

__all__ = ["layer_norm", "layer_norm_backward", "rms_norm", "rms_norm_backward", "linear_cross_entropy",
           "linear_cross_entropy_grad", "grad_norm", "clip_grads", "adamw_state", "adamw_step", "adamw_values", "ADAMW_BLOCK"]

_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _code(what, t):
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: unsupported tensor of dtype {t.dtype} (use float32 or bfloat16)")
    return code


def _on_gpu(what, first, *others):
    """The index of the one GPU that all tensors (None: absent) are on."""
    if not first.is_cuda:
        raise TypeError(f"{what} needs tensors on a ROCm GPU (got {first.device})")
    at = first.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            raise TypeError(f"{what} needs all tensors on one GPU (got {first.device} and {t.device})")
    return at


def _rows(what, name, x):
    """x as a 2-D tensor whose rows are contiguous (copied if they are not),
    and its row stride."""
    if x.dim() == 1:
        x = x.unsqueeze(0)
    if x.dim() != 2:
        raise ValueError(f"{what}: expected a 1-D or 2-D {name}, got shape {tuple(x.shape)}")
    R, D = x.shape
    if (D > 1 and x.stride(1) != 1) or (R > 1 and x.stride(0) < D):
        x = x.contiguous()
    return x, (x.stride(0) if R > 1 else D)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream_of(x):
    """The current stream of the GPU that x is on (0 elsewhere: x is refused)."""
    return _raw_stream(x.get_device()) if x.is_cuda else 0


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *_):
        return None


_HERE = _Here()


def _on(index):
    """The GPU of that index as the current one, where it is not."""
    return _HERE if index == _current_device() else torch.cuda.device(index)


def layer_norm(x, weight=None, bias=None, eps=1e-5, dtype=None):
    """(y, mean, rstd): every row of x normalised to mean 0 and variance 1,
    times `weight` plus `bias`.

        mean = sum(x) / D    rstd = 1 / sqrt(sum((x - mean)^2) / D + eps)
        y = (x - mean) * rstd * weight + bias

    x: [R, D] (or [D], one row) float32 or bfloat16, D >= 1; row-strided views
    are read in place.  weight, bias: [D], of one type, or None.  y has x's
    shape and its type, or `dtype` (the fp32 output of `matrix_mul` normalised
    to the bf16 input of the next product).  mean and rstd are float32 [R]
    whatever the types; `layer_norm_backward` takes them.
    """
    return _lib.host().layer_norm(x, weight, bias, eps, dtype, _stream_of(x))


def layer_norm_backward(dy, x, mean, rstd, weight=None, param_grads=True):
    """(dx, dweight, dbias) of `layer_norm` for the gradient dy of its y.

        wdy = dy * weight;  xhat = (x - mean) * rstd
        dx = rstd * (wdy - mean(wdy) - xhat * mean(wdy * xhat))
        dweight = sum over rows of dy * xhat;  dbias = sum over rows of dy

    x, mean, rstd: the forward pass's input and statistics.  dx has dy's shape
    and type; dweight and dbias are float32 [D], added in a fixed order (the
    same bits on every call).  param_grads=False leaves them out (None).
    """
    return _lib.host().layer_norm_backward(dy, x, mean, rstd, weight, param_grads, _stream_of(dy))


def rms_norm(x, weight=None, residual=None, eps=1e-5, dtype=None):
    """(y, h, rstd): every row of h = x + residual divided by its root mean
    square, times `weight`.

        rstd = 1 / sqrt(sum(h^2) / D + eps);  y = h * rstd * weight

    x: [R, D] (or [D], one row) float32 or bfloat16, D >= 1; row-strided views are
    read in place.  weight: [D] or None.  residual: of x's shape, float32 or
    bfloat16, or None; h has its type (the sum is rounded to it before anything
    else is computed) and is x itself where there is none.  y has x's shape and
    its type, or `dtype`.  With dtype float8_e4m3fn or float8_e5m2 y is the 8-bit
    operand of the next `linear_fp8`, a pair (codes [R, D], scales [R, ceil(D /
    128)]): the codes and scales that `quantize_fp8` gives of the float32 y.  rstd
    is float32 [R]; `rms_norm_backward` takes it and h.  The sum of squares is
    float32: it overflows (rstd 0) for rows of a norm above 2^64, and squares of
    values below 2^-75 are lost.
    """
    return _lib.host().rms_norm(x, weight, residual, eps, dtype)


def rms_norm_backward(dy, h, rstd, weight=None, dh=None, weight_grad=True):
    """(dx, dweight) of `rms_norm` for the gradient dy of its y.

        hhat = h * rstd
        dx = rstd * (dy * weight - hhat * mean(dy * weight * hhat)) + dh
        dweight = sum over rows of dy * hhat

    h, rstd: the forward pass's (h is x where it had no residual).  dh: the
    gradient of h from its other reader, the residual stream, of h's shape, or
    None.  dx is the gradient of x and of the residual alike; it has h's shape and
    dh's type, without dh dy's.  dweight is float32 [D], added in a fixed order
    (the same bits on every call); weight_grad=False leaves it out (None).
    """
    return _lib.host().rms_norm_backward(dy, h, rstd, weight, dh, weight_grad)


_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


@lru_cache(4096)
def _ce_plan(device, N, H, V, ldx, ldw, dtype, code, grad, chunk_rows, x_off, w_off):
    """(workspace bytes, counter bytes, configs) of a call on the current GPU,
    `device`; float32 products run the tuned pick of their shapes, as
    `matrix_mul` does.  x_off, w_off: the addresses modulo 16, all of them that
    the C side looks at."""
    ws, cnt, rows = ctypes.c_size_t(0), ctypes.c_size_t(0), ctypes.c_int64(0)

    def ask(configs):
        _lib.check(_lib.lib().tilec_linear_ce_scratch_bytes(
            x_off or 16, w_off or 16, N, H, V, ldx, ldw, dtype, code, grad, chunk_rows, configs, ctypes.byref(ws),
            ctypes.byref(cnt), ctypes.byref(rows)))
        return ws.value, cnt.value, configs

    plan = ask(None)
    R = rows.value
    if dtype != _lib.F32 or R == 0:
        return plan
    picks = [_tuned(R, H, V, "f32", _lib.X2_COL_MAJOR)]
    picks += [_tuned(R, V, H, "f32", 0), _tuned(V, R, H, "f32", _lib.X1_COL_MAJOR)] if grad else [(-1, 0)] * 2
    return ask((ctypes.c_int32 * 6)(*[v for pick in picks for v in pick]))


def _linear_ce(what, x, weight, target, reduction, ignore_index, grad, grad_loss, chunk_rows):
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        raise ValueError(f"{what}: expected x [N, H] and weight [V, H], got shapes {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    N, H = x.shape
    V = weight.shape[0]
    if H == 0 or V == 0:
        raise ValueError(f"{what}: no features or no classes (x {tuple(x.shape)}, weight {tuple(weight.shape)})")
    if tuple(target.shape) != (N,):
        raise ValueError(f"{what}: target has shape {tuple(target.shape)}, expected ({N},)")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{what}: reduction must be one of {sorted(_REDUCTIONS)} (got {reduction!r})")
    if chunk_rows < 0:
        raise ValueError(f"{what}: chunk_rows must be >= 0 (got {chunk_rows})")
    dtype = _code(what, x)
    if weight.dtype != x.dtype:
        raise TypeError(f"{what}: x has dtype {x.dtype}, weight {weight.dtype}")
    if target.dtype != torch.int64:
        raise TypeError(f"{what}: target has dtype {target.dtype}, expected torch.int64")
    at = _on_gpu(what, x, weight, target, grad_loss)
    if grad_loss is not None:
        want = (N,) if reduction == "none" else ()
        if grad_loss.dtype != torch.float32:
            raise TypeError(f"{what}: grad_loss has dtype {grad_loss.dtype}, expected torch.float32")
        if tuple(grad_loss.shape) != want and not (want == () and tuple(grad_loss.shape) == (1,)):
            raise ValueError(f"{what}: grad_loss has shape {tuple(grad_loss.shape)}, expected {want}")
        grad_loss = grad_loss.contiguous()
    x, ldx = _rows(what, "x", x)
    weight, ldw = _rows(what, "weight", weight)
    target = target.contiguous()
    loss = torch.empty((N,) if reduction == "none" else (), dtype=torch.float32, device=x.device)
    dx = torch.empty((N, H), dtype=x.dtype, device=x.device) if grad else None
    dw = torch.empty((V, H), dtype=x.dtype, device=x.device) if grad else None
    code = _REDUCTIONS[reduction]
    with _on(at):
        stream = _raw_stream(at)
        ws, cnt, configs = _ce_plan(at, N, H, V, ldx, ldw, dtype, code, grad, chunk_rows, x.data_ptr() % 16,
                                    weight.data_ptr() % 16)
        scratch = torch.empty(ws, dtype=torch.uint8, device=x.device) if ws else None
        counters = counters_for(x.device, stream, cnt) if cnt else None  # held until all is enqueued
        _lib.check(_lib.lib().tilec_linear_ce(x.data_ptr(), weight.data_ptr(), target.data_ptr(), loss.data_ptr(),
                                              _ptr(grad_loss), _ptr(dx), _ptr(dw), N, H, V, ldx, ldw, dtype, code,
                                              int(ignore_index), grad, chunk_rows, configs, _ptr(scratch), ws,
                                              _ptr(counters), cnt, stream))
    return loss, dx, dw


def linear_cross_entropy(x, weight, target, reduction="mean", ignore_index=-100):
    """Cross entropy of the logits x @ weight.T against `target`, without
    giving out the logits.

        loss_r = log(sum_v exp(logits[r, v])) - logits[r, target_r]

    x [N, H], weight [V, H]: both float32 or both bfloat16 (row-strided views
    are read in place).  target: int64 [N].  Returns float32: the N losses
    (reduction "none"), or their "sum" or "mean" over the rows that count.
    Rows whose target is `ignore_index` do not: their loss is 0, whatever x
    holds there, and a mean over no rows is 0.  A target that is neither that
    nor a class makes its loss NaN (nothing here reads the device back to
    raise for it).

    Of bfloat16 inputs' logits nothing is kept but a maximum and a sum for every
    64 classes of a row; those of float32 inputs are written to a workspace, for
    as many rows at a time as fit 2 GiB.
    """
    return _linear_ce("linear_cross_entropy", x, weight, target, reduction, ignore_index, 0, None, 0)[0]


def linear_cross_entropy_grad(x, weight, target, reduction="mean", ignore_index=-100, grad_loss=None, chunk_rows=0):
    """(loss, dx, dweight): `linear_cross_entropy` with its gradients, in x's
    type, from one pass over the logits.

        d[r, v] = g_r * (softmax(logits)[r, v] - [v = target_r]);  dx = d @ weight;  dweight = d.T @ x

    grad_loss: the gradient of the loss on the GPU, float32: one value for
    "mean" and "sum", [N] for "none"; None: ones.  Ignored rows add nothing
    and get a dx of zeros, whatever x holds there and whatever grad_loss is
    (float32: where weight is finite).

    Of the logits, one 16-bit value each (float32 inputs: 32-bit) is kept for
    a chunk of rows at a time, `chunk_rows` of them, or by default as many as
    fit 2 GiB of workspace; with more than one chunk, dweight is added up in a
    float32 workspace of its size.

    For bfloat16 inputs d itself is rounded to bfloat16 before the products,
    beside the rounding of dx and dweight.
    """
    return _linear_ce("linear_cross_entropy_grad", x, weight, target, reduction, ignore_index, 1, grad_loss,
                      chunk_rows)


_OWN_COUNTERS = {}  # by device index and stream


def _counters(index, stream, nbytes):
    """Zeroed counters that kernels leave zero: the stream's, in no graph, or in a
    capture the graph's own, zeroed in every replay (a graph may be replayed beside
    its stream's other work).  `index`: the current device's."""
    capturing = _stream_captured()
    kept = None if capturing else _OWN_COUNTERS.get((index, stream))
    if kept is None or kept.numel() < nbytes:
        kept = torch.zeros(nbytes if capturing else max(nbytes, 1 << 17), dtype=torch.uint8,
                           device=torch.device("cuda", index))
        if not capturing:
            _OWN_COUNTERS[index, stream] = kept
    return kept


def grad_norm(grads, max_norm=None, grad_scale=None):
    """(norm, scale): the norm of all values of a list of gradients, and the factor
    that clips it to max_norm, each one float32 on the GPU.

        norm = |grad_scale| * sqrt(sum of all g^2)
        scale = grad_scale * min(1, max_norm / (norm + 1e-6))

    `adamw_step` takes the scale as its grad_scale: gradients are clipped without
    being written.  grads: float32 and bfloat16 tensors on one GPU (None: a
    parameter without a gradient), at least one.  max_norm: at least 0; None or
    infinite: no limit.  grad_scale: a float32 value on the GPU that the gradients are to be
    multiplied by in any case (the inverse of a loss's scale), or None.  Squares
    and sums are float64, in a fixed order: nothing overflows, and the same bits
    come out on every call.  An infinite norm gives a scale of 0, a NaN one NaN.
    """
    return _lib.host().grad_norm(grads, max_norm, grad_scale, _counters)


def clip_grads(grads, max_norm, grad_scale=None):
    """The norm of `grad_norm`; the gradients are multiplied in place by its scale
    (not touched where that is 1).  Two of them may not share memory, and a view
    whose values do not lie side by side is refused (ValueError).  To autograd they
    have been modified in place."""
    return _lib.host().clip_grads(grads, max_norm, grad_scale, _counters)


ADAMW_BLOCK = 256  # values per scale of an 8-bit state


def adamw_state(param, bits=32):
    """(exp_avg, exp_avg_sq): the zero states of `adamw_step` for one
    parameter, float32 tensors of its shape, or with bits=8 a (codes, scales)
    pair each: int8 (exp_avg) and uint8 (exp_avg_sq) codes of the parameter's
    shape and one float32 scale per 256 consecutive values."""
    if bits not in (32, 8):
        raise ValueError(f"adamw_state: states have 32 or 8 bits (got {bits})")
    if bits == 32:
        m, v = torch.zeros((2, *param.shape), dtype=torch.float32, device=param.device)
        return m, v
    scales = torch.zeros((2, -(-param.numel() // ADAMW_BLOCK)), dtype=torch.float32, device=param.device)
    return ((torch.zeros(param.shape, dtype=torch.int8, device=param.device), scales[0]),
            (torch.zeros(param.shape, dtype=torch.uint8, device=param.device), scales[1]))


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               grad_scale=None, copies=None):
    """One AdamW step over lists of tensors, in place.

        g = grad * grad_scale;  p = p * (1 - lr * weight_decay)
        m = beta1 * m + (1 - beta1) * g;  v = beta2 * v + (1 - beta2) * g^2
        p = p - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)

    params: contiguous float32 or bfloat16 tensors; grads: float32 or bfloat16,
    one of each parameter's size (None: that parameter and its states stay as
    they are).  exp_avg, exp_avg_sq (m, v): a state of each parameter, all as
    `adamw_state` makes them, 32-bit or 8-bit (codes, scales).  step counts
    from 1.  grad_scale: a float32 value on the GPU that multiplies every
    gradient (a clipping coefficient).  copies: bfloat16 tensors that get the
    new parameters, rounded (None, or None for some: none).  What is written may
    not overlap anything else in the lists (ValueError), but a result may go
    where it was read from.  All arithmetic is float32; many tensors share a
    launch.  To autograd, what is written has been
    modified in place: a backward pass through a graph that saved a parameter
    before the step raises.

    `step`, `lr` and the other numbers are read on the host: a HIP graph of this
    call repeats the step it was recorded with, bias correction included.
    """
    if step < 1:
        raise ValueError(f"adamw_step: steps count from 1 (got {step})")
    _lib.host().adamw_step(params, grads, exp_avg, exp_avg_sq, copies, step, lr, betas[0], betas[1], eps, weight_decay,
                           grad_scale, _raw_stream)


def adamw_values(states):
    """The float32 values that a list of 8-bit states, (codes, scales) pairs of
    `adamw_step`, stand for: a flat tensor each."""
    packed = _lib.host().adamw_values_table(states)
    if packed is None:
        return []
    table, count, device, out = packed
    with _on(device):
        _lib.check(_lib.lib().tilec_adamw_values(table, count, _raw_stream(device)))
    return out
