"""Paths of the operators behind a forest's leaves that only large calls take, each with a look at the kernels that ran:
leaf numbers kept for the sort, classes in pieces, units of several column tiles, the largest tiles.  A rule that moves
away from a size here fails here.

Tolerances as in test_gpu_leaf_model.py."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_leaf_model import (ACT, EVAL, HALVES, SLOPE, STEP, class_case, complete_forest, draw_ids, grown, near,  # noqa: F401
                                       no_wait_gave_up, normal, plain_loss, strided, table_rows)
from tests.test_gpu_leaf_products import class_gradients_are_near
from treebeard_b200 import leaf_model as lm

pytestmark = pytest.mark.gpu
ONE, PAIR, TALL = 0, 1, 2    # 128 x 128, 256 x 256, 512 x 256


def ran(call):
    """Names of the kernels that a call launches, in order, as far as a profiler tells."""
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    names = [e.name for e in p.events() if "tb::" in e.name]
    if not names:
        pytest.skip("the profiler sees no kernels here")
    return [n.split("(")[0].replace("void tb::", "").replace("tb::", "") for n in names]


def shapes(names, end):
    """Tile shapes of the products that `end` finishes."""
    return [int(n.split(",")[1]) for n in names if n.startswith("tb_dense_kernel<") and end in n]


LEAF = [(25001, 90, 5, 40, torch.bfloat16), (70001, 33, 6, 50, torch.float32), (40000, 60, 7, 31, torch.float16), (150000, 15, 11, 8, torch.bfloat16)]


def leaf_case(n, trees, levels, width, dtype):
    forest, _ = grown(trees, levels, leaf_p=0.1)
    ids = draw_ids(forest, n, blank=0.05)
    return lm.LeafMap(forest), forest, ids, normal(n, width, dtype=dtype, seed=1)


def check_leaf_gradient(back, leaves, rows, grad):
    n, trees = rows.shape
    want = torch.zeros(leaves.num_rows, grad.shape[1], dtype=torch.float64, device="cuda")
    mass, hits = torch.zeros_like(want), torch.zeros(leaves.num_rows, dtype=torch.float64, device="cuda")
    for t in range(trees):
        live = rows[:, t] >= 0
        want.index_add_(0, rows[live, t], grad.double()[live])
        mass.index_add_(0, rows[live, t], grad.double()[live].abs())
        hits.index_add_(0, rows[live, t], torch.ones(int(live.sum()), dtype=torch.float64, device="cuda"))
    near(back, want, hits[:, None] * STEP * mass)


@pytest.mark.parametrize("n,trees,levels,width,dtype", LEAF)
def test_leaf_gradient_with_kept_numbers(n, trees, levels, width, dtype):
    leaves, forest, ids, grad = leaf_case(n, trees, levels, width, dtype)
    back = lm.leaf_sum_backward(leaves, ids, grad)
    check_leaf_gradient(back, leaves, table_rows(forest, ids), grad)
    wide = torch.full((n, trees + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, 1:trees + 1] = ids
    assert torch.equal(lm.leaf_sum_backward(leaves, wide[:, 1:trees + 1], grad), back)
    assert torch.equal(lm.leaf_sum_backward(leaves, ids, strided(grad, 5)), back)


def wide_case():
    trees, levels, n = 3, 16, 700001
    leaves = lm.LeafMap(complete_forest(trees, levels))
    g = torch.Generator(device="cuda").manual_seed(0)
    leaf = torch.randint(0, 1 << levels, (n, trees), device="cuda", generator=g)
    leaf[::7] = (1 << levels) - 1          # number 65535: no mark of two-byte numbers
    return leaves, leaf, (leaf + (1 << levels) - 1).int(), normal(n, 12, dtype=torch.bfloat16)


def test_leaf_gradient_with_kept_four_byte_numbers():
    leaves, leaf, ids, grad = wide_case()
    gone = torch.rand(leaf.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.02
    ids[gone] = 5
    rows = torch.where(gone, -1, leaf + (torch.arange(leaf.shape[1], device="cuda") << 16))
    check_leaf_gradient(lm.leaf_sum_backward(leaves, ids, grad), leaves, rows, grad)


def test_leaf_gradient_at_the_end_of_looked_up_ids():
    """One row below and above the number of ids up to which the sort looks them up itself: the same bits."""
    leaves, forest, ids, grad = leaf_case(65537, 32, 4, 24, torch.float16)
    backs = [lm.leaf_sum_backward(leaves, ids[:n], grad[:n]) for n in (65536, 65537)]
    grad[65536] = 0
    assert torch.equal(lm.leaf_sum_backward(leaves, ids, grad), backs[0])
    check_leaf_gradient(backs[0], leaves, table_rows(forest, ids[:65536]), grad[:65536])


def test_kernels_of_the_leaf_gradient():
    for case in LEAF:
        leaves, _, ids, grad = leaf_case(*case)
        names = ran(lambda: lm.leaf_sum_backward(leaves, ids, grad))
        assert [n.split("<")[0] for n in names] == ["tb_leaf_numbers_kernel", "tb_leaf_grad_kernel"]
        assert "unsigned short" in names[0] and "unsigned short" in names[1]
    leaves, _, ids, grad = wide_case()
    names = ran(lambda: lm.leaf_sum_backward(leaves, ids, grad))
    assert len(names) == 2 and all("unsigned int" in n for n in names)
    names = ran(lambda: lm.leaf_sum_backward(leaves, ids[:600], grad[:600]))
    assert len(names) == 1 and "int>" in names[0] and "unsigned" not in names[0]


# rows, width, classes; pieces of the classes; tiles of the scores in loss and (a piece each) in the gradient; column
# tiles of a unit
CLASS = [(6000, 777, 9001, 1, TALL, [TALL], 1), (8200, 700, 20011, 2, PAIR, [PAIR, TALL], 4), (14000, 100, 20011, 3, PAIR, [PAIR] * 3, 7),
         (33000, 24, 8200, 3, PAIR, [PAIR] * 3, 7), (5000, 1030, 30011, 2, TALL, [PAIR, TALL], 1), (8190, 1024, 32700, 2, TALL, [TALL] * 2, 3)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,width,classes", [c[:3] for c in CLASS])
def test_class_loss_of_large_calls(n, width, classes, dtype):
    x, w, b, labels = class_case(n, width, classes, dtype)
    z, lse, loss, live, at = plain_loss(x, w, b, labels)
    off = torch.cat([((width + 4) * STEP * (x[a:a + 2048].double().abs() @ w.double().abs().t() + z[a:a + 2048].abs())).max(1).values for a in range(0, n, 2048)])
    off = off + (600 + classes / 64) * STEP + 8 * STEP * (z.abs().max(1).values + 1)
    got, got_lse = lm.class_loss(x, w, labels, b)
    near(got_lse, lse, off)
    near(got, loss, 2 * off)
    weights = (torch.rand(n, device="cuda") + 0.5) / n
    outs = lm.class_loss_backward(weights, x, w, labels, got_lse, b)
    class_gradients_are_near(outs, x, w, b, labels, weights, z, got_lse, live, at)
    assert all(torch.equal(p, q) for p, q in zip(outs, lm.class_loss_backward(weights, x, w, labels, got_lse, b)))


@pytest.mark.parametrize("n,width,classes,pieces,loss_shape,grad_shapes,run", CLASS)
def test_kernels_of_large_class_losses(n, width, classes, pieces, loss_shape, grad_shapes, run):
    dtype = torch.bfloat16
    x, w, b, labels = class_case(n, width, classes, dtype)
    assert shapes(ran(lambda: lm.class_loss(x, w, labels, b)), "LseEnd") == [loss_shape]
    lse, weights = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    names = ran(lambda: lm.class_loss_backward(weights, x, w, labels, lse, b))
    assert shapes(names, "ScoreGradEnd") == grad_shapes and len(grad_shapes) == pieces
    # what a row keeps of its scores tells how many column tiles (256 wide) a unit has
    units = -(-(-(-classes // 256)) // run)
    size = lm._size("tbk_class_loss_workspace", n, width, classes, 2, 1, 0)
    up = lambda v: -(-v // 256) * 256
    assert size == up(n * 4 * units * 8) + up(n * 4)


def test_tiles_of_large_layers():
    """512 x 256 tiles with an activation, the value before it and a residual, and in a backward pass."""
    for dtype in HALVES:
        n, inputs, outputs = 33000, 600, 2500
        x, w = normal(n, inputs, dtype=dtype), normal(outputs, inputs, dtype=dtype, scale=inputs ** -0.5, seed=1)
        b, r = normal(outputs, dtype=dtype, seed=2), normal(n, outputs, dtype=dtype, seed=3)
        z, mass = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t()
        off = (inputs + 2) * STEP * (mass + z.abs())
        got, pre = lm.linear(x, w, b, "relu", r, keep_pre=True)
        near(pre, z, off)
        near(got, ACT["relu"][0](z) + r.double(), off + EVAL * (z.abs() + r.double().abs()))
        assert torch.equal(lm.linear(x, w, b, "relu", r), got)
        assert shapes(ran(lambda: lm.linear(x, w, b, "relu", r, keep_pre=True)), "ResultEnd") == [TALL]
    x, w, g = normal(9000, 1000, dtype=dtype), normal(5000, 1000, dtype=dtype, seed=1), normal(9000, 5000, dtype=dtype, seed=2)
    names = ran(lambda: lm.linear_backward(g, x, w))
    assert shapes(names, "ResultEnd") == [TALL] and names[-1].startswith("tb_dense_finish_kernel")
    dx, dw, db = lm.linear_backward(g, x, w)
    G, X, W = g.double(), x.double(), w.double()
    near(dx, G @ W, 5002 * STEP * (G.abs() @ W.abs()))
    near(dw, G.t() @ X, 9002 * STEP * (G.abs().t() @ X.abs()))
    near(db, G.sum(0), 9002 * STEP * G.abs().sum(0))


@pytest.mark.parametrize("dtype", HALVES)
def test_a_model_of_many_rows_with_weights_of_ones(dtype):
    """What fp16 asks for at training batches: gradients of the sum, whose size the type holds."""
    n, classes = 20000, 700
    forest, marg = grown(30, 5)
    rows = torch.from_numpy(marg.sample_rows(np.random.default_rng(0), n)).cuda()
    params = dict(table=normal(lm.LeafMap(forest).num_rows, 48, dtype=dtype, scale=30 ** -0.5), w1=normal(96, 48, dtype=dtype, scale=48 ** -0.5, seed=1),
                  w2=normal(96, 96, dtype=dtype, scale=96 ** -0.5, seed=3), wc=normal(classes, 96, dtype=dtype, scale=96 ** -0.5, seed=4),
                  bc=normal(classes, dtype=dtype, scale=0.1, seed=5))
    model = lm.LeafModel(forest, params["table"], [(params["w1"], None, "gelu", False), (params["w2"], None, "silu", True)], params["wc"], params["bc"])
    labels = torch.arange(n, device="cuda") * 13 % classes
    loss, grads = model.loss_and_grads(rows, labels, torch.ones(n, device="cuda"))
    q = {k: v.double().requires_grad_(True) for k, v in params.items()}
    h = q["table"][table_rows(forest, model.forest.predict_leaf_ids(rows))].sum(1)
    h = ACT["gelu"][0](h @ q["w1"].t())
    h = ACT["silu"][0](h @ q["w2"].t()) + h
    z = h @ q["wc"].t() + q["bc"]
    want = torch.logsumexp(z, 1) - z.gather(1, labels[:, None])[:, 0]
    want.sum().backward()
    # (the roundings of a chain, as in the smaller model's test: 8 half steps in the 2-norm)
    half = torch.finfo(dtype).eps / 2
    assert (loss.double() - want).norm() <= 8 * half * want.norm()
    got = dict(table=grads["table"], w1=grads["layers"][0][0], w2=grads["layers"][1][0], wc=grads["weight"], bc=grads["bias"])
    for k in q:
        assert (got[k].double() - q[k].grad).norm() <= 8 * half * q[k].grad.norm(), k
