"""The operators behind a forest's leaves, as far as they go without a GPU: symbols, refusals, sizes."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_abi import declared
from treebeard_b200 import _lib, kernels, leaf_model as lm, synth

INVALID, UNSUPPORTED = 1, 3


def refused(status, text=None):
    class Check:
        def __enter__(self):
            self.catch = pytest.raises(kernels.TbkError, match=text)
            self.info = self.catch.__enter__()

        def __exit__(self, *a):
            done = self.catch.__exit__(*a)
            assert self.info.value.status == status
            return done
    return Check()


def test_every_declared_symbol_is_exported_and_bound():
    names = declared("tbk_leaf.h", "TBK_EXPORT")
    assert len(names) == 16 and len(set(names)) == 16
    for name in names:
        assert getattr(lm.lib(), name).argtypes is not None


def test_leaf_map_refuses_malformed_forests():
    forest = synth.generate_forest(0, 5, 4, 8, 0.1, 0.1, synth.Marginal("normal", 8))
    c, keep = kernels.forest_arrays_c(forest)
    out = ctypes.c_void_p()
    create = lm.lib().tbk_leaf_map_create
    assert create(ctypes.byref(c), 0, None) == INVALID
    assert create(None, 0, ctypes.byref(out)) == INVALID
    c.num_trees = 0
    assert create(ctypes.byref(c), 0, ctypes.byref(out)) == INVALID
    c, keep = kernels.forest_arrays_c(forest)
    keep[0][3] = keep[0][2]
    assert create(ctypes.byref(c), 0, ctypes.byref(out)) == INVALID and b"tree 2" in lm.lib().tbk_last_error()
    forest = synth.generate_forest(0, 5, 4, 8, 0.1, 0.1, synth.Marginal("normal", 8))
    c, keep = kernels.forest_arrays_c(forest)
    keep[1][keep[0][3]:keep[0][4]] = 0
    assert create(ctypes.byref(c), 0, ctypes.byref(out)) == INVALID and b"tree 3 has no leaf" in lm.lib().tbk_last_error()
    assert out.value is None and lm.lib().tbk_leaf_map_rows(None) == -1 and lm.lib().tbk_leaf_map_free(None) == 0


def test_the_library_checks_its_own_arguments():
    """No device is touched before the arguments hold: made-up addresses are never followed."""
    L, p = lm.lib(), 1 << 20
    err = lambda: L.tbk_last_error().decode()
    assert L.tbk_leaf_sum(None, p, 1, 1, p, 1, 1, 0, p, 1, None, 0, None) == INVALID
    assert L.tbk_leaf_sum_backward(None, p, 1, 1, p, 1, 1, 0, p, 1, p, 4, None) == INVALID

    def linear(x=p, ld_x=8, w=p, act=0, out=p, n=4, inputs=8, outputs=4, kind=2):
        return L.tbk_linear(x, ld_x, w, inputs, None, act, None, 0, out, outputs, None, 0, n, inputs, outputs, kind, None, 0, 0, None)
    assert linear(kind=0) == UNSUPPORTED and "16-bit" in err()
    assert linear(kind=7) == INVALID and linear(n=-1) == INVALID and linear(inputs=0) == INVALID and linear(outputs=0) == INVALID
    assert linear(n=1 << 40) == UNSUPPORTED
    assert linear(x=None) == INVALID and "x is null" in err()
    assert linear(w=None) == INVALID and linear(out=None) == INVALID
    assert linear(ld_x=7) == INVALID and "row to row" in err()
    assert linear(act=4) == INVALID and linear(act=-1) == INVALID
    assert linear(n=0) == 0    # nothing to do

    def back(pre=p, act=1, ws=p, size=1 << 40):
        return L.tbk_linear_backward(p, 4, p, 8, p, 8, pre, 4, act, None, 0, p, 8, p, 8, p, 4, 8, 4, 2, ws, size, 0, None)
    # (a made-up device: what passes the checks ends there)
    assert back(pre=None) == INVALID and "pre is null" in err()
    assert back(ws=None) == INVALID and "workspace" in err()
    assert back(size=1) == INVALID and back(ws=p + 8) == INVALID and "aligned" in err()

    def loss(labels=p, label_bytes=8, classes=100, out=p, ws=p):
        return L.tbk_class_loss(p, 8, p, 8, None, labels, label_bytes, out, p, 4, 8, classes, 1, ws, 1 << 40, 0, None)
    assert loss(labels=None) == INVALID and loss(label_bytes=2) == INVALID and loss(classes=0) == INVALID
    assert loss(out=None) == INVALID and loss(ws=None) == INVALID

    def loss_back(grad=p, lse=p):
        return L.tbk_class_loss_backward(grad, p, 8, p, 8, None, p, 8, lse, p, 8, p, 8, None, 4, 8, 100, 1, p, 1 << 40, 0, None)
    assert loss_back(grad=None) == INVALID and loss_back(lse=None) == INVALID


def test_workspaces_grow_with_the_call_and_stay_bounded():
    def size(name, n, k, m):
        out = ctypes.c_uint64()
        assert getattr(lm.lib(), name + "_workspace")(n, k, m, 2, 1, 0, ctypes.byref(out)) == 0
        return out.value
    # the scores of this call would take 8 GiB in fp32; neither direction keeps them
    assert size("tbk_class_loss", 16384, 256, 131072) < 1 << 28
    assert size("tbk_class_loss_backward", 16384, 256, 131072) < 1 << 29
    assert size("tbk_linear_backward", 1000, 64, 64) >= 1000 * 64 * 2
    for name in ("tbk_linear", "tbk_linear_backward", "tbk_class_loss", "tbk_class_loss_backward"):
        assert getattr(lm.lib(), name + "_workspace")(1, 1, 1, 2, 1, 0, None) == INVALID


def _map(rows=12, trees=3):
    """What the shape checks look at, without a device."""
    return SimpleNamespace(num_rows=rows, num_trees=trees, device=0, _h=None)


def test_shapes_and_types_are_refused_before_any_launch():
    t = lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=dtype)
    ids = torch.zeros(4, 3, dtype=torch.int32)
    with refused(INVALID, "table"):
        lm.leaf_sum(_map(), ids, t(11, 8))
    with refused(INVALID, "ids"):
        lm.leaf_sum(_map(), ids.long(), t(12, 8))
    with refused(INVALID, "ids"):
        lm.leaf_sum(_map(), ids[:, :2], t(12, 8))
    with refused(INVALID, "no type"):
        lm.leaf_sum(_map(), ids, t(12, 8, dtype=torch.float64))
    with refused(INVALID, "row have to lie"):
        lm.leaf_sum(_map(), ids, t(8, 12).t())
    with refused(INVALID, "grad"):
        lm.leaf_sum_backward(_map(), ids, t(5, 8))
    with refused(UNSUPPORTED, "16-bit"):
        lm.linear(t(4, 8, dtype=torch.float32), t(5, 8, dtype=torch.float32))
    with refused(INVALID, "does not take"):
        lm.linear(t(4, 8, dtype=torch.float64), t(5, 8))
    with refused(INVALID, "weight"):
        lm.linear(t(4, 8), t(5, 7))
    with refused(INVALID, "weight"):
        lm.linear(t(4, 8), t(5, 8, dtype=torch.float16))
    with refused(INVALID, "bias"):
        lm.linear(t(4, 8), t(5, 8), t(4))
    with refused(INVALID, "residual"):
        lm.linear(t(4, 8), t(5, 8), residual=t(4, 8))
    with refused(INVALID, "activation"):
        lm.linear(t(4, 8), t(5, 8), activation="tanh")
    with refused(INVALID, "needs the values"):
        lm.linear_backward(t(4, 5), t(4, 8), t(5, 8), activation="gelu")
    with refused(INVALID, "skip"):
        lm.linear_backward(t(4, 5), t(4, 8), t(5, 8), skip=t(4, 5))
    with refused(INVALID, "labels"):
        lm.class_loss(t(4, 8), t(5, 8), torch.zeros(4, dtype=torch.int16))
    with refused(INVALID, "labels"):
        lm.class_loss(t(4, 8), t(5, 8), torch.zeros(5, dtype=torch.int64))
    with refused(INVALID, "lse"):
        lm.class_loss_backward(torch.zeros(4), t(4, 8), t(5, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(3))
    with refused(INVALID, "grad_loss"):
        lm.class_loss_backward(t(4), t(4, 8), t(5, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4))


def test_host_tensors_are_refused():
    t = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16)
    with refused(INVALID, "CUDA device"):
        lm.linear(t(4, 8), t(5, 8))
    with refused(INVALID, "CUDA device"):
        lm.class_loss(t(4, 8), t(5, 8), torch.zeros(4, dtype=torch.int64))
    with refused(INVALID, "CUDA device"):
        lm.leaf_sum(_map(), torch.zeros(4, 3, dtype=torch.int32), t(12, 8))
    with refused(INVALID, "CUDA device"):
        lm.LeafModel(None, t(12, 8), [], t(5, 8))


def test_overlap_is_seen_by_bytes():
    a = torch.zeros(100)
    lm._apart("out", a[:50], a[50:], None)
    lm._apart("out", a[:0], a)
    with refused(INVALID, "overlaps"):
        lm._apart("out", a[:51], a[50:])
    m = torch.zeros(10, 8)
    with refused(INVALID, "overlaps"):   # columns of one matrix interlace
        lm._apart("out", m[:, :4], m[:, 4:])


def test_a_closed_leaf_map_is_refused():
    leaves = lm.LeafMap.__new__(lm.LeafMap)
    leaves._h, leaves._size = None, lambda *a: 0   # (as if it held a handle)
    leaves.close()
    with refused(INVALID, "closed"):
        leaves._size("tbk_leaf_sum_workspace", 1, 8, 0)


def test_a_stream_of_another_device_is_refused():
    other = SimpleNamespace(device=torch.device("cuda", 1))
    tensor = SimpleNamespace(is_cuda=True, get_device=lambda: 0)
    called = []
    call = lm._on_stream(lambda *a, **k: called.append(a))
    with refused(INVALID, "stream"):
        call(None, _like(tensor), stream=other)
    with refused(INVALID, "stream"):
        call(None, bias=_like(tensor), stream=other)
    assert not called


def _like(fake):
    class Tensor(torch.Tensor):
        get_device = staticmethod(fake.get_device)
    return torch.zeros(1).as_subclass(Tensor)


def test_more_trees_than_a_launch_reaches_are_refused():
    forest = synth.generate_forest(0, 5, 4, 8, 0.1, 0.1, synth.Marginal("normal", 8))
    c, keep = kernels.forest_arrays_c(forest)
    out = ctypes.c_void_p()
    c.num_trees = 65535 * 32 + 1   # (refused before an array is read)
    assert lm.lib().tbk_leaf_map_create(ctypes.byref(c), 0, ctypes.byref(out)) == UNSUPPORTED
    assert b"2097120 trees" in lm.lib().tbk_last_error()


def test_tensors_without_dimensions_are_refused():
    leaves = SimpleNamespace(_h=1, device=0, num_trees=3, num_rows=12)
    with refused(INVALID):
        lm.leaf_sum_backward(leaves, torch.zeros((), dtype=torch.int32), torch.zeros(2, 8))
    with refused(INVALID):
        lm.leaf_sum_backward(leaves, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(()))
