"""Gradients of the operators behind a forest's leaves against differences of the plain forms in 64 bits, along the
gradient's own signs: there the difference is the sum of the gradient's magnitudes, and a gradient that is zero, negated
or of a wrong size is far outside the bound."""
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_leaf_model import ACT, HALVES, STEP, class_case, complete_forest, no_wait_gave_up, normal, plain_loss  # noqa: F401
from treebeard_b200 import leaf_model as lm

pytestmark = pytest.mark.gpu


def slope(value, args, k, d, h):
    up, down = [list(args) for _ in range(2)]
    up[k], down[k] = args[k] + h * d, args[k] - h * d
    return (value(*up) - value(*down)) / (2 * h)


def agree(value, args, k, got, want, off, h=1e-5):
    """got: the kernel's gradient of argument k; want: its formula in 64 bits; off: bound of every element's error."""
    d = want.sign()
    mass, bound = want.abs().sum(), off.sum()
    there = slope(value, args, k, d, h)
    assert (there - mass).abs() <= 1e-4 * mass      # (the formula is the difference's)
    assert bound <= mass / 5                        # (the bound can tell)
    assert ((got.double() * d).sum() - there).abs() <= bound + 1e-4 * mass


# the largest second derivative of an activation
CURVE = {"identity": 0.0, "gelu": 0.8, "silu": 0.5}


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("name", CURVE)
@pytest.mark.parametrize("n,inputs,outputs", [(40, 24, 56), (300, 64, 130)])
def test_layer(n, inputs, outputs, name, dtype):
    x, w, b = normal(n, inputs, dtype=dtype), normal(outputs, inputs, dtype=dtype, scale=0.2, seed=1), normal(outputs, dtype=dtype, seed=2)
    g = normal(n, outputs, dtype=dtype, seed=3)
    pre = lm.linear(x, w, b, name, keep_pre=True)[1]
    got = lm.linear_backward(g, x, w, pre, name)
    args = [t.double() for t in (x, w, b)]
    G = g.double()
    z = args[0] @ args[1].t() + args[2]
    dz = G * ACT[name][1](z)
    # the kept value and dz are each rounded once, the result too; fp32 sums and slopes stay below a hundredth of that
    half = torch.finfo(dtype).eps / 2 * 1.02
    kept = half * G.abs() * CURVE[name] * z.abs()
    off = kept + half * dz.abs()
    value = lambda x, w, b: (G * ACT[name][0](x @ w.t() + b)).sum()
    for k, (want, o) in enumerate(((dz @ args[1], off @ args[1].abs()), (dz.t() @ args[0], off.t() @ args[0].abs()), (dz.sum(0), kept.sum(0)))):
        agree(value, args, k, got[k], want, o + half * want.abs())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,width,classes", [(40, 24, 30), (200, 72, 255)])
def test_class_loss(n, width, classes, dtype):
    x, w, b, labels = class_case(n, width, classes, dtype)
    weights = torch.rand(n, device="cuda") + 0.5
    lse = lm.class_loss(x, w, labels, b)[1]
    got = lm.class_loss_backward(weights, x, w, labels, lse, b)
    args = [t.double() for t in (x, w, b)]
    z, exact, _, live, at = plain_loss(x, w, b, labels)
    p = torch.exp(z - exact[:, None]).scatter_add_(1, at[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
    dz = p * torch.where(live, weights.double(), 0.0)[:, None]
    half = torch.finfo(dtype).eps / 2 * 1.02
    off = half * dz.abs() + 2.0 ** -37 * weights.max().double()
    value = lambda x, w, b: (weights.double() * plain_loss(x, w, b, labels)[2]).sum()
    for k, (want, o) in enumerate(((dz @ args[1], off @ args[1].abs()), (dz.t() @ args[0], off.t() @ args[0].abs()), (dz.sum(0), 1e-4 * dz.abs().sum(0)))):
        agree(value, args, k, got[k], want, o + half * want.abs())


@pytest.mark.parametrize("dtype", [torch.float32] + HALVES)
def test_leaf_sum(dtype):
    trees, levels, n, width = 12, 4, 500, 40
    leaves = lm.LeafMap(complete_forest(trees, levels))
    g = torch.Generator(device="cuda").manual_seed(0)
    leaf = torch.randint(0, 1 << levels, (n, trees), device="cuda", generator=g)
    rows = leaf + (torch.arange(trees, device="cuda") << levels)
    table, grad = normal(leaves.num_rows, width, dtype=dtype), normal(n, width, dtype=dtype, seed=1)
    got = lm.leaf_sum_backward(leaves, (leaf + (1 << levels) - 1).int(), grad)
    G = grad.double()
    want = torch.zeros(leaves.num_rows, width, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want)
    for t in range(trees):
        want.index_add_(0, rows[:, t], G)
        mass.index_add_(0, rows[:, t], G.abs())
    off = n * STEP * mass + torch.finfo(dtype).eps / 2 * want.abs()
    agree(lambda table: (table[rows].sum(1) * G).sum(), [table.double()], 0, got, want, off)
