"""Language-model operators on device arrays: scores of tokens, distillation from a teacher's top
logits, the gated linear recurrence, and their gradients.

They stand beside the front end's `nn.log_softmax`, `nn.cross_entropy_loss` and `Tensor.cumsum`
(`crates/nn/src/functional/activation.rs:174-187`, `loss.rs:32-65`, `src/lowerer/lower.rs:691-735`; the
reference has none of them) and run as hand-written kernels through the C ABI of
`include/eclat_hip.h`, which defines every argument, special value and refusal.

An array is a `HipBuffer` with a shape and a dtype, a `View` into one, or any object with the
attributes of a torch tensor on the same GPU (`data_ptr()`, `shape`, `stride()`, `dtype`, `get_device()`).  Work is
queued on the device handle's stream: for arrays of another library open the handle on the stream
that this library works on, `HipDevice(index, stream=...)`.

    dev = HipDevice(0, stream=torch.cuda.current_stream().cuda_stream)
    scores = token_logprobs(dev, logits, targets, top=5, out=Logprobs(logp, entropy, norm, top_logp, top_ids))
    grad = token_logprobs_backward(dev, logits, targets, norm, entropy, grad_logp, grad_entropy, out=grad)

Without `out` the results are new `HipBuffer`s.  Nothing waits for the GPU.

Tensors of another library are memory to these calls: none of them is recorded for that library's differentiation
(a tensor that requires a gradient is read like any other, and gets none from here; each call's gradient is its `_backward`),
and what is written to `out` is not counted as a change of it.  The calls do not keep a tensor alive for work that is queued.
"""

from __future__ import annotations

import struct
from collections import namedtuple
from typing import Optional, Sequence

from ._lib import check, lib
from .backend import HipBuffer, HipDevice
from .frontend.ast import F32, I32, DType

__all__ = ["Logprobs", "Distilled", "ScanGrads", "View", "token_logprobs", "token_logprobs_backward", "token_logprobs_workspace",
           "distill_loss", "distill_loss_backward", "distill_loss_workspace", "gated_scan", "gated_scan_backward",
           "gated_scan_workspace", "gated_scan_backward_workspace", "MAX_TOP", "MAX_TEACHER"]

MAX_TOP = 32             # alternatives a row can report
MAX_TEACHER = 1024       # tokens a teacher can name in a row

Logprobs = namedtuple("Logprobs", "logp entropy norm top_logp top_ids")
Distilled = namedtuple("Distilled", "loss norm grad")
ScanGrads = namedtuple("ScanGrads", "grad_gate grad_x grad_state")

_CODES = {"float32": 0, "f32": 0, "bfloat16": 1, "bf16": 1, "float16": 2, "f16": 2, "int32": 3, "i32": 3, "int64": 4, "i64": 4}
_ITEM = (4, 2, 2, 4, 8)
_DTYPES = (F32, DType("bf16"), DType("f16"), I32, DType("i64"))
_known = {}              # dtype object -> code
_NONE = (0, 0, 0, 0, 0, 0)

_A = "QQQqqq"
_SCORE = struct.Struct("=qqqqd" + 8 * _A)
_SCORE_GRAD = struct.Struct("=qqqd" + 7 * _A)
_DISTILL = struct.Struct("=qqqd" + 8 * _A)
_SCAN = struct.Struct("=qqqq" + 7 * _A)
_SCAN_GRAD = struct.Struct("=qqqq" + 10 * _A)


class View:
    """A part of a `HipBuffer`: `shape` elements of `dtype` from byte `offset` on, contiguous unless
    `strides` (in elements) say otherwise."""

    def __init__(self, buffer: HipBuffer, shape: Sequence[int], dtype: DType, offset: int = 0, strides: Optional[Sequence[int]] = None):
        self.buffer, self.shape, self.dtype, self.offset = buffer, tuple(int(s) for s in shape), dtype, int(offset)
        self.strides = _dense(self.shape) if strides is None else tuple(int(s) for s in strides)
        if len(self.strides) != len(self.shape):
            raise ValueError("a view has as many strides as axes")

    def stride(self):
        return self.strides


def _dense(shape):
    out, n = [], 1
    for s in reversed(shape):
        out.append(n)
        n *= s
    return tuple(reversed(out))


def _code(dtype, name):
    code = _CODES.get(str(dtype).rsplit(".", 1)[-1])
    if code is None:
        raise TypeError(f"{name}: element type {dtype} is not supported")
    _known[dtype] = code
    return code


def _array(device, x, name, ndim, want=None):
    """(shape, element type, fields of an eh_array) of an array; `want`: the shape it has to have."""
    try:
        address, shape, strides = x.data_ptr(), x.shape, x.stride()
        index, dtype = x.get_device(), x.dtype
    except AttributeError:
        return _buffer_array(device, x, name, ndim, want)
    if index != device.index:
        raise ValueError(f"{name}: lives on " + ("the host" if index < 0 else f"GPU {index}") + f", the handle is of GPU {device.index}")
    code = _known.get(dtype)
    if code is None:
        code = _code(dtype, name)
    s0, s1, last = _layout(name, shape, strides, ndim, want)
    if last <= 0:                                    # an empty tensor has no address
        return shape, code, (0, 16, 0, s0, s1, code)
    return shape, code, (0, address, last * _ITEM[code], s0, s1, code)


def _buffer_array(device, x, name, ndim, want):
    buf = x.buffer if isinstance(x, View) else x
    if not isinstance(buf, HipBuffer):
        raise TypeError(f"{name}: a {type(x).__name__} is no array on the device")
    if buf.device is not device:
        raise ValueError(f"{name}: lives on another device handle")
    if x.dtype is None:
        raise TypeError(f"{name}: the buffer has no element type")
    code = _known.get(x.dtype)
    if code is None:
        code = _code(x.dtype, name)
    shape = tuple(x.shape)
    strides, offset = (_dense(shape), 0) if buf is x else (x.strides, x.offset)
    if offset < 0:
        raise ValueError(f"{name}: starts before its buffer")
    s0, s1, _ = _layout(name, shape, strides, ndim, want)
    return shape, code, (buf._h.value, offset, 0, s0, s1, code)


def _layout(name, shape, strides, ndim, want):
    """The outer strides, and how many elements lie between the first and the last."""
    if want is not None and shape != want or len(shape) != ndim:
        raise ValueError(f"{name}: shape {tuple(shape)}, expected " + (f"{ndim} axes" if want is None else str(tuple(want))))
    n = shape[-1]
    if n > 1 and strides[-1] != 1:
        raise ValueError(f"{name}: " + ("has to be contiguous" if ndim == 1 else "the last axis has to be contiguous"))
    if ndim == 1:
        return 1, 0, n
    if ndim == 2:
        return strides[0], 0, (shape[0] - 1) * strides[0] + n if n and shape[0] else 0
    return strides[0], strides[1], (shape[0] - 1) * strides[0] + (shape[1] - 1) * strides[1] + n if n and shape[0] and shape[1] else 0


def _small(device, x, name, want, code):
    """A contiguous array of one type; None: absent."""
    if x is None:
        return _NONE
    _, got, fields = _array(device, x, name, len(want), want)
    if got != code:
        raise TypeError(f"{name}: has to be {_DTYPES[code]}")
    if len(want) == 2 and want[0] > 1 and fields[3] != want[1]:
        raise ValueError(f"{name}: has to be contiguous")
    return fields


def _workspace(device, x):
    if x is None:
        return _NONE
    if isinstance(x, HipBuffer):
        if x.device is not device:
            raise ValueError("workspace: lives on another device handle")
        return (x._h.value, 0, 0, 0, 0, 0)
    if x.get_device() != device.index or not x.is_contiguous():
        raise ValueError("workspace: has to be contiguous memory of the handle's GPU")
    return (0, x.data_ptr(), x.numel() * x.element_size(), 0, 0, 0)


def _new(device, shape, code):
    return HipBuffer(device, shape, _DTYPES[code])


def _bytes_needed(fn, device, packed):
    import ctypes
    n = ctypes.c_size_t()
    check(fn(device._h, packed, ctypes.byref(n)))
    return n.value


# ---- scores of tokens -------------------------------------------------------------------------------


def token_logprobs(device: HipDevice, logits, targets, *, top: int = 0, entropy: bool = True, scale: float = 1.0,
                   ignore_index: int = -1, out: Optional[Logprobs] = None, workspace=None) -> Logprobs:
    """Log probability of one given token for each row of `logits` [rows, vocab] under
    softmax(scale * logits), the entropy, and the `top` likeliest tokens with theirs.  `out.norm` is what
    `token_logprobs_backward` reads."""
    shape, code, z = _array(device, logits, "logits", 2)
    rows, vocab = shape
    _, _, t = _array(device, targets, "targets", 1, (rows,))
    if out is None:
        out = Logprobs(_new(device, [rows], 0), _new(device, [rows], 0) if entropy else None, _new(device, [rows, 2], 0),
                       _new(device, [rows, top], 0) if top else None, _new(device, [rows, top], 3) if top else None)
    if top and (out.top_logp is None or out.top_ids is None):
        raise ValueError("top_logp, top_ids: needed where alternatives are asked for")
    packed = _SCORE.pack(rows, vocab, top, ignore_index, scale, *z, *t,
                         *_small(device, out.logp, "logp", (rows,), 0), *_small(device, out.entropy, "entropy", (rows,), 0),
                         *_small(device, out.norm, "norm", (rows, 2), 0),
                         *(_small(device, out.top_logp, "top_logp", (rows, top), 0) if top else _NONE),
                         *(_small(device, out.top_ids, "top_ids", (rows, top), 3) if top else _NONE), *_workspace(device, workspace))
    check(lib.eh_token_logprobs(device._h, packed, 0))
    return out


def token_logprobs_workspace(device: HipDevice, logits, *, top: int = 0) -> int:
    """Bytes `token_logprobs` works in besides its arrays; needed as `workspace` under stream capture."""
    shape, _, z = _array(device, logits, "logits", 2)
    return _bytes_needed(lib.eh_token_logprobs_workspace, device, _SCORE.pack(*shape, top, 0, 1.0, *z, *(7 * _NONE)))


def token_logprobs_backward(device: HipDevice, logits, targets, norm, entropy=None, grad_logp=None, grad_entropy=None, *,
                            scale: float = 1.0, ignore_index: int = -1, out=None):
    """Gradient of sum(grad_logp * logp + grad_entropy * entropy) with respect to the logits, in their type.
    `norm` (and, with `grad_entropy`, `entropy`) as `token_logprobs` returned them."""
    shape, code, z = _array(device, logits, "logits", 2)
    rows, vocab = shape
    _, _, t = _array(device, targets, "targets", 1, (rows,))
    if grad_entropy is not None and entropy is None:
        raise ValueError("entropy: needed for its gradient")
    if out is None:
        out = _new(device, [rows, vocab], code)
    packed = _SCORE_GRAD.pack(rows, vocab, ignore_index, scale, *z, *t, *_small(device, norm, "norm", (rows, 2), 0),
                              *_small(device, entropy, "entropy", (rows,), 0), *_small(device, grad_logp, "grad_logp", (rows,), 0),
                              *_small(device, grad_entropy, "grad_entropy", (rows,), 0),
                              *_array(device, out, "out", 2, (rows, vocab))[2])
    check(lib.eh_token_logprobs_backward(device._h, packed, 0))
    return out


# ---- distillation -----------------------------------------------------------------------------------


def _distill(device, logits, teacher_logits, teacher_ids, row_weight, temperature, loss, norm, grad, workspace):
    shape, code, z = _array(device, logits, "logits", 2)
    rows, vocab = shape
    tshape, _, t = _array(device, teacher_logits, "teacher_logits", 2)
    if tshape[0] != rows:
        raise ValueError(f"teacher_logits: {tshape[0]} rows, the logits have {rows}")
    _, _, i = _array(device, teacher_ids, "teacher_ids", 2, tuple(tshape))
    return _DISTILL.pack(rows, vocab, tshape[1], temperature, *z, *t, *i, *_small(device, row_weight, "row_weight", (rows,), 0),
                         *_small(device, loss, "loss", (rows,), 0), *_small(device, norm, "norm", (rows, 2), 0),
                         *(_NONE if grad is None else _array(device, grad, "grad", 2, (rows, vocab))[2]), *_workspace(device, workspace))


def distill_loss(device: HipDevice, logits, teacher_logits, teacher_ids, *, temperature: float = 1.0, row_weight=None,
                 grad: bool = False, out: Optional[Distilled] = None, workspace=None) -> Distilled:
    """temperature^2 KL(teacher || student) of each row: the student's softmax(logits / temperature) over the
    vocabulary, the teacher's softmax over the tokens `teacher_ids` [rows, k] (negative: no entry) with
    `teacher_logits`.  With `grad` the gradient of sum(row_weight * loss) with respect to the logits as well."""
    if out is None:
        shape, code, _ = _array(device, logits, "logits", 2)
        out = Distilled(_new(device, [shape[0]], 0), _new(device, [shape[0], 2], 0), _new(device, shape, code) if grad else None)
    if grad and out.grad is None:
        raise ValueError("grad: needed where the gradient is asked for")
    packed = _distill(device, logits, teacher_logits, teacher_ids, row_weight, temperature, out.loss, out.norm,
                      out.grad if grad else None, workspace)
    check(lib.eh_distill_loss(device._h, packed, 0))
    return out


def distill_loss_workspace(device: HipDevice, logits) -> int:
    """Bytes `distill_loss` works in besides its arrays; needed as `workspace` under stream capture."""
    shape, _, z = _array(device, logits, "logits", 2)
    return _bytes_needed(lib.eh_distill_loss_workspace, device, _DISTILL.pack(*shape, 1, 1.0, *z, *(7 * _NONE)))


def distill_loss_backward(device: HipDevice, logits, teacher_logits, teacher_ids, norm, grad_loss=None, *,
                          temperature: float = 1.0, out=None):
    """Gradient of sum(grad_loss * loss) with respect to the logits (`grad_loss` None: ones), from `distill_loss`'s norm."""
    if out is None:
        shape, code, _ = _array(device, logits, "logits", 2)
        out = _new(device, shape, code)
    packed = _distill(device, logits, teacher_logits, teacher_ids, grad_loss, temperature, None, norm, out, None)
    check(lib.eh_distill_loss_backward(device._h, packed, 0))
    return out


# ---- gated linear recurrence ------------------------------------------------------------------------


def gated_scan(device: HipDevice, gate, x, *, state=None, lengths=None, log_gate: bool = False, out=None, final=None,
               workspace=None):
    """h_t = a_t h_(t-1) + x_t along axis 1 of [batch, time, width], with a = gate or exp(gate); h_(-1) is `state`
    [batch, width] (f32) or 0.  `final` receives h of the last step in f32: the next call's `state`, which makes a call
    with time 1 a decoding step.  `lengths` [batch] (i32): steps behind them are neither read nor written, so that `out` holds there what it held (a new one:
    zeros).  Returns `out`."""
    shape, code, g = _array(device, gate, "gate", 3)
    shape = tuple(shape)
    batch, time, width = shape
    if out is None:
        out = _new(device, shape, code)
    packed = _SCAN.pack(batch, time, width, bool(log_gate), *g, *_array(device, x, "x", 3, shape)[2],
                        *_small(device, state, "state", (batch, width), 0), *_small(device, lengths, "lengths", (batch,), 3),
                        *_array(device, out, "out", 3, shape)[2], *_small(device, final, "final", (batch, width), 0),
                        *_workspace(device, workspace))
    check(lib.eh_gated_scan(device._h, packed, 0))
    return out


def gated_scan_workspace(device: HipDevice, gate) -> int:
    """Bytes `gated_scan` works in besides its arrays; needed as `workspace` under stream capture."""
    shape, _, g = _array(device, gate, "gate", 3)
    return _bytes_needed(lib.eh_gated_scan_workspace, device, _SCAN.pack(*shape, 0, *g, *(6 * _NONE)))


def gated_scan_backward(device: HipDevice, gate, h, grad_h, *, state=None, lengths=None, log_gate: bool = False,
                        grad_final=None, out: Optional[ScanGrads] = None, workspace=None) -> ScanGrads:
    """Gradients of `gated_scan` with respect to gate, x and (where there is one) state, from its outputs `h` and
    their gradient `grad_h` (and the final states', `grad_final`)."""
    shape, code, g = _array(device, gate, "gate", 3)
    shape = tuple(shape)
    batch, time, width = shape
    if out is None:
        out = ScanGrads(_new(device, shape, code), _new(device, shape, code), None if state is None else _new(device, [batch, width], 0))
    packed = _SCAN_GRAD.pack(batch, time, width, bool(log_gate), *g, *_array(device, h, "h", 3, shape)[2],
                             *_array(device, grad_h, "grad_h", 3, shape)[2], *_small(device, state, "state", (batch, width), 0),
                             *_small(device, lengths, "lengths", (batch,), 3),
                             *_small(device, grad_final, "grad_final", (batch, width), 0),
                             *_array(device, out.grad_gate, "grad_gate", 3, shape)[2], *_array(device, out.grad_x, "grad_x", 3, shape)[2],
                             *_small(device, out.grad_state, "grad_state", (batch, width), 0), *_workspace(device, workspace))
    check(lib.eh_gated_scan_backward(device._h, packed, 0))
    return out


def gated_scan_backward_workspace(device: HipDevice, gate) -> int:
    """Bytes `gated_scan_backward` works in besides its arrays; needed as `workspace` under stream capture."""
    shape, _, g = _array(device, gate, "gate", 3)
    return _bytes_needed(lib.eh_gated_scan_backward_workspace, device, _SCAN_GRAD.pack(*shape, 0, *g, *(9 * _NONE)))


# ---- the front end's calls ----------------------------------------------------------------------------


def run(device: HipDevice, name: str, attrs: dict, inputs, outputs):
    """An operator node of a graph: `inputs` (buffer, shape, dtype), dense; `outputs` (shape, dtype).  Returns the
    outputs' buffers."""
    ins = [View(b, shape, dtype) for b, shape, dtype in inputs]
    outs = [HipBuffer(device, shape, dtype) for shape, dtype in outputs]
    if name == "token_logprobs":
        token_logprobs(device, *ins, out=Logprobs(*outs, None, None), **attrs)
    elif name == "token_logprobs_backward":
        logits, targets, norm, entropy, *grads = ins
        g = grads.pop(0) if attrs["logp"] else None
        e = grads.pop(0) if attrs["entropy"] else None
        token_logprobs_backward(device, logits, targets, norm, entropy, g, e, scale=attrs["scale"],
                                ignore_index=attrs["ignore_index"], out=outs[0])
    elif name == "distill_loss":
        distill_loss(device, *ins, out=Distilled(*outs, None), **attrs)
    elif name == "distill_loss_backward":
        distill_loss_backward(device, *ins, out=outs[0], **attrs)
    elif name == "gated_scan":
        gated_scan(device, *ins[:2], state=ins[2] if len(ins) > 2 else None, out=outs[0], **attrs)
    elif name == "gated_scan_backward":
        gated_scan_backward(device, *ins[:3], state=ins[3] if len(ins) > 3 else None,
                            out=ScanGrads(*outs, *[None] * (3 - len(outs))), **attrs)
    else:
        raise ValueError(f"no operator '{name}'")
    return outs
