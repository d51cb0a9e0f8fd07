"""A second model on a forest's leaf indices: the operators of include/tbk_leaf.h for callers that hold
torch CUDA tensors, and a model that chains them.

``DeviceForest.predict_leaf_ids`` says which leaf every row reached in every tree.  ``leaf_sum`` turns
that into a dense row (one embedding per leaf, summed over the trees), ``linear`` is a layer with bias,
activation and residual, ``class_loss`` the softmax cross entropy over as many classes as one likes (the
scores are never stored).  Each has its gradient as a call of its own; the calls take part in no autograd
graph.  All of them are ordered by the current stream of the tensors' device, or by ``stream``, and can be
captured into a CUDA graph; a workspace, where one is needed, comes from torch's allocator on that stream.
With ``stream`` the arguments may be given up right after the call; results belong to that stream, and whoever uses
them on another waits for it first.

The reference ends at the forest's own prediction and has no counterpart.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import kernels
from .kernels import TbkError, _stream_ptr

ACTIVATIONS = {"identity": 0, "relu": 1, "gelu": 2, "silu": 3}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INVALID, _UNSUPPORTED = 1, 3
_lib = None


def lib():
    global _lib
    if _lib is None:
        L = kernels.lib()
        vp, i64, i32, u64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_uint64
        size = ctypes.POINTER(u64)
        L.tbk_leaf_map_create.argtypes = [vp, i32, ctypes.POINTER(vp)]
        L.tbk_leaf_map_free.argtypes = [vp]
        L.tbk_leaf_map_rows.argtypes = [vp]
        L.tbk_leaf_map_rows.restype = i64
        L.tbk_leaf_sum_workspace.argtypes = [vp, i64, i64, i32, size]
        L.tbk_leaf_sum.argtypes = [vp, vp, i64, i64, vp, i64, i64, i32, vp, i64, vp, u64, vp]
        L.tbk_leaf_sum_backward_workspace.argtypes = [vp, i64, i64, i32, size]
        L.tbk_leaf_sum_backward.argtypes = [vp, vp, i64, i64, vp, i64, i64, i32, vp, i64, vp, u64, vp]
        for name in ("tbk_linear", "tbk_linear_backward", "tbk_class_loss", "tbk_class_loss_backward"):
            getattr(L, name + "_workspace").argtypes = [i64, i64, i64, i32, i32, i32, size]
        L.tbk_leaf_check_status.argtypes = [i32]
        L.tbk_linear.argtypes = [vp, i64, vp, i64, vp, i32, vp, i64, vp, i64, vp, i64, i64, i64, i64, i32, vp, u64, i32, vp]
        L.tbk_linear_backward.argtypes = [vp, i64, vp, i64, vp, i64, vp, i64, i32, vp, i64, vp, i64, vp, i64, vp, i64, i64,
                                          i64, i32, vp, u64, i32, vp]
        L.tbk_class_loss.argtypes = [vp, i64, vp, i64, vp, vp, i32, vp, vp, i64, i64, i64, i32, vp, u64, i32, vp]
        L.tbk_class_loss_backward.argtypes = [vp, vp, i64, vp, i64, vp, vp, i32, vp, vp, i64, vp, i64, vp, i64, i64, i64,
                                              i32, vp, u64, i32, vp]
        _lib = L
    return _lib


def _check(rc):
    if rc:
        raise TbkError(rc, lib().tbk_last_error().decode())


def _refuse(message):
    raise TbkError(_INVALID, message)


def _matrix(name, t, dtype, rows=None, cols=None):
    """Checks a row-major matrix; returns its row stride."""
    shape = t.shape
    if len(shape) != 2 or t.dtype is not dtype:
        _refuse(f"{name}: a 2-d tensor of {dtype} is wanted, not {t.dim()}-d of {t.dtype}")
    n, m = shape
    if (rows is not None and n != rows) or (cols is not None and m != cols):
        _refuse(f"{name} has shape ({n}, {m}), wanted are ({'any' if rows is None else rows}, {'any' if cols is None else cols})")
    ld, step = t.stride()
    if ld >= m and (step == 1 or m == 1):
        return ld
    if n and ((step != 1 and m > 1) or (ld < m and n > 1)):
        _refuse(f"{name}: the elements of a row have to lie one behind the other, the rows apart")
    return m


def _vector(name, t, dtype, length):
    if t.shape != (length,) or t.dtype is not dtype:
        _refuse(f"{name}: {length} elements of {dtype} are wanted, not {tuple(t.shape)} of {t.dtype}")
    if length > 1 and t.stride(0) != 1:
        _refuse(f"{name}: the elements have to lie one behind the other")


def _device(first, *tensors):
    """Number of the CUDA device that all tensors lie on."""
    index = first.get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        _refuse("all tensors have to be on one CUDA device")
    return index


def _half(t, what):
    kind = _TYPES.get(t.dtype)
    if kind == 0:
        raise TbkError(_UNSUPPORTED, f"{what} takes 16-bit floating point types (fp16, bf16)")
    if kind is None:
        _refuse(f"{what} does not take {t.dtype}")
    return kind


def _span(t):
    """First and last byte + 1 that a tensor touches."""
    a = t.data_ptr()
    return a, a + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else a


def _apart(name, out, *inputs):
    a, b = _span(out)
    for t in inputs:
        if t is not None:
            c, d = _span(t)
            if a < d and c < b:
                _refuse(f"{name} overlaps another tensor of the call")


def _on_stream(call):
    """``stream=`` of a call: the stream that its work is ordered by and its own memory comes from."""
    @functools.wraps(call)
    def wrapper(*args, stream=None, **kwargs):
        if stream is None:
            return call(*args, **kwargs)
        tensors = [t for t in (*args, *kwargs.values()) if isinstance(t, torch.Tensor)]
        for t in tensors:
            if t.get_device() != stream.device.index:
                _refuse(f"the stream is on {stream.device}, a tensor of the call is not")
        with torch.cuda.stream(stream):
            result = call(*args, **kwargs)
        for t in tensors:   # (memory that its owner gives back meanwhile is not handed out before the work is done)
            t.record_stream(stream)
        return result
    return wrapper


@functools.lru_cache(maxsize=1024)
def _size(function, *sizes):
    """Bytes of a call's workspace: a function of its sizes alone."""
    need = ctypes.c_uint64()
    _check(getattr(lib(), function)(*sizes, ctypes.byref(need)))
    return need.value


def _workspace(like, size):
    """(tensor to keep until the call returns, its address)"""
    if not size:
        return None, None
    ws = like.new_empty(size, dtype=torch.uint8)
    return ws, ws.data_ptr()


def _readable(x, ld_x, weight, ld_w):
    """Whether the kernels read x and weight where they are: rows that begin at multiples of 16 bytes."""
    return int(not (x.data_ptr() | weight.data_ptr()) & 15 and (ld_x % 8 == 0 or x.shape[0] <= 1) and (ld_w % 8 == 0 or weight.shape[0] <= 1))


def check_status(device: int = 0):
    """Waits for the device (all of its streams); raises TbkError if a bounded wait inside one of these kernels gave up
    since the last check.  The status is the device's and is cleared by the check: of several threads, the first to ask
    learns of it."""
    _check(lib().tbk_leaf_check_status(device))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _closed(*_):
    _refuse("the leaf map is closed")


class LeafMap:
    """Which row of an embedding table each leaf of a forest stands for: the leaves of all trees, numbered
    tree by tree in node order (``num_rows`` of them).  ``forest`` is any object with the flat forest
    attributes (those that ``DeviceForest`` takes)."""

    def __init__(self, forest, device: int = 0):
        c, keep = kernels.forest_arrays_c(forest)
        h = ctypes.c_void_p()
        _check(lib().tbk_leaf_map_create(ctypes.byref(c), device, ctypes.byref(h)))
        self._h = h
        self.device = device
        self.num_trees = len(keep[0]) - 1
        self.num_rows = int(lib().tbk_leaf_map_rows(h))
        self._size = functools.lru_cache(maxsize=256)(lambda function, *sizes: _size.__wrapped__(function, h, *sizes))

    def close(self):
        if getattr(self, "_h", None):
            try:
                lib().tbk_leaf_map_free(self._h)
            except TypeError:      # interpreter shutdown: module globals are already gone
                pass
        self._h = None
        self._size = _closed       # (what was there holds the handle)

    __del__ = close


def _leaf_call(leaves, ids, other, what):
    ld = _matrix("ids", ids, torch.int32, None, leaves.num_trees)
    kind = _TYPES.get(other.dtype)
    if kind is None:
        _refuse(f"{what}: {other.dtype} is no type of an embedding table")
    device = _device(ids, other)
    if device != leaves.device:
        _refuse(f"the leaf map is on device {leaves.device}, the tensors on {device}")
    return ld, device, kind


@_on_stream
def leaf_sum(leaves: LeafMap, ids, table, out=None):
    """out[n] = sum over trees of the table row of the leaf that row n reached.  ids: int32 [n, trees] as
    predict_leaf_ids gives them; an id that is no leaf of its tree (-1 for a padded row) adds nothing.
    table: [leaves.num_rows, width], fp32, fp16 or bf16.  Returns [n, width] of table's type."""
    ld_table = _matrix("table", table, table.dtype, leaves.num_rows)
    ld_ids, device, kind = _leaf_call(leaves, ids, table, "leaf_sum")
    n, width = ids.shape[0], table.shape[1]
    if out is None:
        out, ld_out = table.new_empty((n, width)), width
    else:
        ld_out = _matrix("out", out, table.dtype, n, width)
        _device(ids, out)
        _apart("out", out, ids, table)
    L = lib()
    size = leaves._size("tbk_leaf_sum_workspace", n, width, kind)
    keep, ws = _workspace(table, size)
    _check(L.tbk_leaf_sum(leaves._h, ids.data_ptr(), n, ld_ids, table.data_ptr(), ld_table, width, kind, out.data_ptr(), ld_out,
                          ws, size, _stream_ptr(None, device)))
    return out


@_on_stream
def leaf_sum_backward(leaves: LeafMap, ids, grad, out=None):
    """Gradient of leaf_sum with respect to the table, [leaves.num_rows, width] of grad's type, from grad
    [n, width], the gradient of its result."""
    ld_grad = _matrix("grad", grad, grad.dtype, ids.shape[0] if ids.dim() else None)
    ld_ids, device, kind = _leaf_call(leaves, ids, grad, "leaf_sum_backward")
    n, width = grad.shape
    if out is None:
        out, ld_out = grad.new_empty((leaves.num_rows, width)), width
    else:
        ld_out = _matrix("out", out, grad.dtype, leaves.num_rows, width)
        _device(ids, out)
        _apart("out", out, ids, grad)
    L = lib()
    size = leaves._size("tbk_leaf_sum_backward_workspace", n, width, kind)
    keep, ws = _workspace(grad, size)
    _check(L.tbk_leaf_sum_backward(leaves._h, ids.data_ptr(), n, ld_ids, grad.data_ptr(), ld_grad, width, kind, out.data_ptr(), ld_out,
                                   ws, size, _stream_ptr(None, device)))
    return out


@_on_stream
def linear(x, weight, bias=None, activation: str = "identity", residual=None, keep_pre: bool = False, out=None):
    """activation(x weight^T + bias) + residual.  x [n, inputs], weight [outputs, inputs], bias [outputs],
    residual [n, outputs], all fp16 or all bf16; activation: identity, relu, gelu (by the normal
    distribution's integral) or silu.  Returns [n, outputs]; with keep_pre also the value before the
    activation, which linear_backward takes.  out may be residual."""
    kind = _half(x, "linear")
    dtype = x.dtype
    ld_x = _matrix("x", x, dtype)
    n, inputs = x.shape
    ld_w = _matrix("weight", weight, dtype, None, inputs)
    outputs = weight.shape[0]
    if bias is not None:
        _vector("bias", bias, dtype, outputs)
    ld_r = _matrix("residual", residual, dtype, n, outputs) if residual is not None else 0
    act = ACTIVATIONS.get(activation)
    if act is None:
        _refuse(f"unknown activation {activation!r}")
    device = _device(x, weight, bias, residual)
    if out is None:
        out, ld_o = x.new_empty((n, outputs)), outputs
    else:
        ld_o = _matrix("out", out, dtype, n, outputs)
        _device(x, out)
        same = residual is not None and out.data_ptr() == residual.data_ptr() and ld_o == ld_r
        _apart("out", out, x, weight, bias, None if same else residual)
    pre = x.new_empty((n, outputs)) if keep_pre else None
    L = lib()
    size = _size("tbk_linear_workspace", n, inputs, outputs, kind, _readable(x, ld_x, weight, ld_w), device)
    keep, ws = _workspace(x, size)
    _check(L.tbk_linear(x.data_ptr(), ld_x, weight.data_ptr(), ld_w, _ptr(bias), act, _ptr(residual), ld_r, out.data_ptr(), ld_o,
                        _ptr(pre), outputs, n, inputs, outputs, kind, ws, size, device, _stream_ptr(None, device)))
    return (out, pre) if keep_pre else out


@_on_stream
def linear_backward(grad, x, weight, pre=None, activation: str = "identity", bias: bool = True, skip=None):
    """Gradients of linear from grad, the gradient of its result (which is the residual's gradient too):
    (of x, of weight) and, with ``bias``, of the bias.  pre is what linear kept; identity needs none.
    skip [n, inputs] is added to x's gradient: grad itself, where x was the residual too.
    grad times the activation's slope is rounded to the type before the products: in fp16 it should lie between
    6e-5 and 65504, so scale the loss."""
    kind = _half(x, "linear_backward")
    dtype = x.dtype
    ld_x = _matrix("x", x, dtype)
    n, inputs = x.shape
    ld_w = _matrix("weight", weight, dtype, None, inputs)
    outputs = weight.shape[0]
    ld_g = _matrix("grad", grad, dtype, n, outputs)
    act = ACTIVATIONS.get(activation)
    if act is None:
        _refuse(f"unknown activation {activation!r}")
    if pre is None and act:
        _refuse(f"{activation} needs the values before the activation (pre)")
    ld_p = _matrix("pre", pre, dtype, n, outputs) if pre is not None else 0
    ld_s = _matrix("skip", skip, dtype, n, inputs) if skip is not None else 0
    device = _device(grad, x, weight, pre, skip)
    grad_x, grad_w = x.new_empty((n, inputs)), x.new_empty((outputs, inputs))
    grad_b = x.new_empty(outputs) if bias else None
    L = lib()
    size = _size("tbk_linear_backward_workspace", n, inputs, outputs, kind, _readable(x, ld_x, weight, ld_w), device)
    keep, ws = _workspace(x, size)
    _check(L.tbk_linear_backward(grad.data_ptr(), ld_g, x.data_ptr(), ld_x, weight.data_ptr(), ld_w, _ptr(pre), ld_p, act, _ptr(skip),
                                 ld_s, grad_x.data_ptr(), inputs, grad_w.data_ptr(), inputs, _ptr(grad_b), n, inputs, outputs, kind,
                                 ws, size, device, _stream_ptr(None, device)))
    return (grad_x, grad_w, grad_b) if bias else (grad_x, grad_w)


def _class_call(what, x, weight, labels, bias):
    kind = _half(x, what)
    ld_x = _matrix("x", x, x.dtype)
    n, width = x.shape
    ld_w = _matrix("weight", weight, x.dtype, None, width)
    classes = weight.shape[0]
    if labels.dtype is not torch.int64 and labels.dtype is not torch.int32:
        _refuse(f"labels are int64 or int32, not {labels.dtype}")
    _vector("labels", labels, labels.dtype, n)
    if bias is not None:
        _vector("bias", bias, x.dtype, classes)
    return kind, ld_x, ld_w, n, width, classes


@_on_stream
def class_loss(x, weight, labels, bias=None):
    """Softmax cross entropy over the classes with scores z = x weight^T + bias, which are never stored.
    x [n, width], weight [classes, width], bias [classes], all fp16 or all bf16; labels [n], int64 or int32:
    a label outside 0 .. classes-1 leaves its row out (loss 0).  Returns fp32 (loss [n], lse [n]) with
    lse = log sum exp z."""
    kind, ld_x, ld_w, n, width, classes = _class_call("class_loss", x, weight, labels, bias)
    device = _device(x, weight, labels, bias)
    loss, lse = x.new_empty(n, dtype=torch.float32), x.new_empty(n, dtype=torch.float32)
    L = lib()
    size = _size("tbk_class_loss_workspace", n, width, classes, kind, _readable(x, ld_x, weight, ld_w), device)
    keep, ws = _workspace(x, size)
    _check(L.tbk_class_loss(x.data_ptr(), ld_x, weight.data_ptr(), ld_w, _ptr(bias), labels.data_ptr(), labels.element_size(),
                            loss.data_ptr(), lse.data_ptr(), n, width, classes, kind, ws, size, device, _stream_ptr(None, device)))
    return loss, lse


@_on_stream
def class_loss_backward(grad_loss, x, weight, labels, lse, bias=None):
    """Gradients of sum(grad_loss * loss) with respect to x, weight and, where one is given, bias.
    grad_loss: fp32 [n], every row's weight in the objective (1/n for the mean); lse: what class_loss gave.  Rows without
    a label add nothing, provided that x is finite there (zero times a NaN is one, in weight's gradient)."""
    kind, ld_x, ld_w, n, width, classes = _class_call("class_loss_backward", x, weight, labels, bias)
    _vector("grad_loss", grad_loss, torch.float32, n)
    _vector("lse", lse, torch.float32, n)
    device = _device(x, weight, labels, bias, grad_loss, lse)
    grad_x, grad_w = x.new_empty((n, width)), x.new_empty((classes, width))
    grad_b = x.new_empty(classes) if bias is not None else None
    L = lib()
    size = _size("tbk_class_loss_backward_workspace", n, width, classes, kind, _readable(x, ld_x, weight, ld_w), device)
    keep, ws = _workspace(x, size)
    _check(L.tbk_class_loss_backward(grad_loss.data_ptr(), x.data_ptr(), ld_x, weight.data_ptr(), ld_w, _ptr(bias), labels.data_ptr(),
                                     labels.element_size(), lse.data_ptr(), grad_x.data_ptr(), width, grad_w.data_ptr(), width,
                                     _ptr(grad_b), n, width, classes, kind, ws, size, device, _stream_ptr(None, device)))
    return (grad_x, grad_w, grad_b) if bias is not None else (grad_x, grad_w)


class LeafModel:
    """rows -> leaves -> sum of embeddings -> linear layers -> classes.

    forest: flat forest arrays; they are packed for the device here, with ``schedule`` as DeviceForest
    takes it.  table: [leaves, width]; layers: (weight, bias or None, activation, add the layer's input)
    for each layer; weight, bias: of the classes.  All parameters are fp16 or all bf16 CUDA tensors, kept
    by reference: an optimiser updates them in place."""

    def __init__(self, forest, table, layers, weight, bias=None, batch_hint: int = 0, **schedule):
        device = _device(table, weight, bias, *(t for l in layers for t in l[:2]))
        self.forest = kernels.DeviceForest(forest, device=device, batch_hint=batch_hint, **(schedule or {"representation": "auto"}))
        self.leaves = LeafMap(forest, device)
        self.table, self.layers, self.weight, self.bias = table, list(layers), weight, bias
        width = table.shape[1]
        for w, _, _, add in self.layers:
            if w.shape[1] != width or (add and w.shape[0] != width):
                _refuse(f"a layer of {tuple(w.shape)}{' with its input added' if add else ''} cannot follow {width} columns")
            width = w.shape[0]
        if weight.shape[1] != width:
            _refuse(f"the classes' weight has {weight.shape[1]} columns, the layers end in {width}")

    def features(self, rows, kept=None):
        """What the classes' scores are products of: [n, width].  rows: CUDA float32 [n, F]."""
        ids = self.forest.predict_leaf_ids(rows)
        h = leaf_sum(self.leaves, ids, self.table)
        if kept is not None:
            kept.append(ids)
        for weight, bias, activation, add in self.layers:
            x = h
            h = linear(x, weight, bias, activation, x if add else None, keep_pre=kept is not None and activation != "identity")
            pre = None
            if isinstance(h, tuple):
                h, pre = h
            if kept is not None:
                kept.append((x, pre))
        return h

    def scores(self, rows):
        """The classes' scores [n, classes], stored: for prediction, where a few rows are looked at."""
        return linear(self.features(rows), self.weight, self.bias)

    def loss(self, rows, labels):
        """Every row's softmax cross entropy, fp32 [n]."""
        return class_loss(self.features(rows), self.weight, labels, self.bias)[0]

    def loss_and_grads(self, rows, labels, row_weights=None):
        """(loss [n], gradients of sum(row_weights * loss)); row_weights: fp32 [n], 1/n each if None.
        Gradients: {"table", "layers": [(weight, bias or None)], "weight", "bias" or None}, of the parameters' type, as
        are those between the layers.  fp16 has few digits below 6e-5, where weights of 1/n lead with thousands of rows:
        pass larger ones (ones, say) and divide in the optimiser.  bf16 needs no scale."""
        kept = []
        h = self.features(rows, kept)
        loss, lse = class_loss(h, self.weight, labels, self.bias)
        if row_weights is None:
            row_weights = torch.full_like(loss, 1.0 / max(1, len(loss)))
        g, grad_w, *grad_b = class_loss_backward(row_weights, h, self.weight, labels, lse, self.bias)
        layers = []
        for (weight, bias, activation, add), (x, pre) in zip(reversed(self.layers), reversed(kept[1:])):
            g, gw, *gb = linear_backward(g, x, weight, pre, activation, bias=bias is not None, skip=g if add else None)
            layers.append((gw, gb[0] if gb else None))
        return loss, {"table": leaf_sum_backward(self.leaves, kept[0], g), "layers": layers[::-1], "weight": grad_w,
                      "bias": grad_b[0] if grad_b else None}
