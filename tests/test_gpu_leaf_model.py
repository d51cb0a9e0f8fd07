"""The operators behind a forest's leaves against plain 64-bit forms of their formulas.

Tolerances, elementwise, from the arithmetic: an output is rounded once (half a step, eps / 2 relative, of
its type; in fp16 half of 2^-24 below the normal range); a sum of K fp32 terms is off by at most K steps of
2^-23 of the sum of their magnitudes, in whatever order and whether additions round or truncate; operands
that are rounded to 16 bits before a product (dz of the backward passes) bring eps / 2 of every term."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from treebeard_b200 import kernels, leaf_model as lm, synth

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]
STEP = 2.0 ** -23


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    lm.check_status(0)


def rounding(want, dtype):
    return torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype is torch.float16 else 0.0)


def near(got, want, extra):
    """|got - want| <= rounding of got's type + extra; equal where want is not finite.  A value of half a step or more
    above the type's largest number rounds to infinity (65504 + 16 in fp16, whose step there is 32)."""
    assert got.shape == want.shape
    kind = torch.finfo(got.dtype)
    beyond = want.abs() + extra >= kind.max * (1 + kind.eps / 4)
    want = torch.where(beyond & torch.isinf(got) & (got.sign() == want.sign()), got.double(), want)
    odd = ~torch.isfinite(want)
    assert torch.equal(got[odd].double().nan_to_num(7e300), want[odd].nan_to_num(7e300))
    err = torch.where(odd, 0.0, (got.double() - want).abs())
    over = torch.where(odd, 0.0, err - rounding(want, got.dtype) * 1.0001 - extra)
    assert (over <= 0).all(), f"off by up to {over.max().item():.3g} beyond the bound, error {err.max().item():.3g}"


def normal(*shape, dtype=torch.float32, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def strided(t, pad):
    """The same values with `pad` foreign elements between the rows (NaN, which no result may show)."""
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def grown(trees, levels, leaf_p=0.2, features=6, seed=3):
    marg = synth.Marginal("normal", features)
    return synth.generate_forest(seed, trees, levels, features, leaf_p, 0.1, marg), marg


def draw_ids(forest, n, seed=0, blank=0.0):
    """Leaves of every tree, drawn unevenly; a share of them struck out."""
    rng = np.random.default_rng(seed)
    ids = np.empty((n, forest.num_trees), np.int32)
    for t in range(forest.num_trees):
        leaves = np.flatnonzero(np.asarray(forest.left[forest.tree_off[t]:forest.tree_off[t + 1]]) < 0)
        ids[:, t] = leaves[(len(leaves) * rng.random(n) ** 3).astype(int)]
    ids[rng.random(ids.shape) < blank] = -1
    return torch.from_numpy(ids).cuda()


def table_rows(forest, ids):
    """Row of the table per (row, tree) by plain numbering; -1 where the id is no leaf."""
    left = np.asarray(forest.left)
    number = np.where(left < 0, np.cumsum(left < 0) - 1, -1)
    ids, off = ids.cpu().numpy().astype(np.int64), np.asarray(forest.tree_off)
    at = ids + off[:-1]
    good = (ids >= 0) & (at < off[1:])
    return torch.from_numpy(np.where(good, number[np.where(good, at, 0)], -1)).cuda()


@pytest.mark.parametrize("dtype", [torch.float32] + HALVES)
@pytest.mark.parametrize("trees,levels,n,width", [(1, 0, 3, 1), (7, 3, 1, 8), (33, 6, 257, 50), (100, 5, 64, 128),
                                                  (257, 4, 30, 264), (12, 9, 1000, 31), (5, 5, 40, 1031)])
def test_leaf_sum_and_its_gradient(trees, levels, n, width, dtype):
    forest, _ = grown(trees, levels)
    leaves = lm.LeafMap(forest)
    assert leaves.num_rows == int((np.asarray(forest.left) < 0).sum())
    ids = draw_ids(forest, n, blank=0.1)
    if n > 3:
        ids[3] = -1                                  # a row without any leaf
        ids[2, 0] = 1 << 30                          # beyond the tree
        ids[1, trees - 1] = 0 if levels else -5      # the root: an inner node, unless it is the only leaf
    rows = table_rows(forest, ids)
    live = rows >= 0
    table, grad = normal(leaves.num_rows, width, dtype=dtype), normal(n, width, dtype=dtype, seed=1)
    picked = torch.where(live[..., None], table.double()[rows.clamp(min=0)], 0.0)
    got = lm.leaf_sum(leaves, ids, table)
    near(got, picked.sum(1), trees * STEP * picked.abs().sum(1))
    if n > 3:
        assert (got[3] == 0).all()

    flat, spread = rows[live], grad.double()[:, None, :].expand(-1, trees, -1)[live]
    want = torch.zeros(leaves.num_rows, width, dtype=torch.float64, device="cuda").index_add_(0, flat, spread)
    mass = torch.zeros_like(want).index_add_(0, flat, spread.abs())
    back = lm.leaf_sum_backward(leaves, ids, grad)
    near(back, want, n * STEP * mass)
    assert torch.equal(back, lm.leaf_sum_backward(leaves, ids, grad))   # no order of its own
    # strides of everything, outputs of the caller's
    out, dout = strided(got * 0, 3), strided(back * 0, 5)
    assert torch.equal(lm.leaf_sum(leaves, ids, strided(table, 1), out=out), got)
    lm.leaf_sum_backward(leaves, ids, strided(grad, 7), out=dout)
    assert torch.equal(dout, back) and out.data_ptr() != got.data_ptr()
    wide_ids = torch.full((n, trees + 2), -1, dtype=torch.int32, device="cuda")
    wide_ids[:, :trees] = ids
    assert torch.equal(lm.leaf_sum(leaves, wide_ids[:, :trees], table), got)
    assert torch.equal(lm.leaf_sum_backward(leaves, wide_ids[:, :trees], grad), back)


@pytest.mark.parametrize("n", [0, 1, 40000, 70001])
def test_leaf_sum_over_the_range_of_rows(n):
    forest, _ = grown(9, 4)
    leaves = lm.LeafMap(forest)
    ids, width = draw_ids(forest, n), 24
    table, grad = normal(leaves.num_rows, width), normal(n, width, seed=1)
    rows = table_rows(forest, ids)
    picked = table.double()[rows]
    near(lm.leaf_sum(leaves, ids, table), picked.sum(1), 9 * STEP * picked.abs().sum(1))
    spread = grad.double()[:, None, :].expand(-1, 9, -1).reshape(-1, width)
    want = torch.zeros(leaves.num_rows, width, dtype=torch.float64, device="cuda").index_add_(0, rows.reshape(-1), spread)
    mass = torch.zeros_like(want).index_add_(0, rows.reshape(-1), spread.abs())
    near(lm.leaf_sum_backward(leaves, ids, grad), want, max(1, n) * STEP * mass)


def test_leaf_gradient_of_one_tree_with_many_leaves():
    forest, _ = grown(2, 13, leaf_p=0.0)
    leaves = lm.LeafMap(forest)
    ids = draw_ids(forest, 3000)
    grad, rows = normal(3000, 16), table_rows(forest, ids)
    spread = grad.double()[:, None, :].expand(-1, 2, -1).reshape(-1, 16)
    want = torch.zeros(leaves.num_rows, 16, dtype=torch.float64, device="cuda").index_add_(0, rows.reshape(-1), spread)
    mass = torch.zeros_like(want).index_add_(0, rows.reshape(-1), spread.abs())
    near(lm.leaf_sum_backward(leaves, ids, grad), want, 3000 * STEP * mass)


ACT = {"identity": (lambda z: z, lambda z: torch.ones_like(z)),
       "relu": (lambda z: z.clamp(min=0), lambda z: (z > 0).double()),
       "gelu": (lambda z: 0.5 * z * (1 + torch.erf(z / 2 ** 0.5)),
                lambda z: 0.5 * (1 + torch.erf(z / 2 ** 0.5)) + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5),
       "silu": (lambda z: z * torch.sigmoid(z), lambda z: torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z))))}
# the slopes of the activations and of their derivatives stay below 1.13 and 0.8; their fp32 evaluation is off by
# a few steps of values that are themselves below |z| + 1
SLOPE, EVAL = 1.13, 16 * STEP

LINEAR = [(1, 1, 1), (1, 1024, 1024), (2, 8, 300), (3, 7, 5), (5, 777, 333), (17, 64, 64), (64, 96, 129), (100, 33, 257),
          (128, 128, 256), (129, 130, 72), (130, 2100, 40), (257, 64, 513), (300, 520, 1), (1000, 16, 24), (700, 200, 1100)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,inputs,outputs", LINEAR)
def test_linear(n, inputs, outputs, dtype):
    x, w = normal(n, inputs, dtype=dtype), normal(outputs, inputs, dtype=dtype, scale=inputs ** -0.5, seed=1)
    b, r = normal(outputs, dtype=dtype, seed=2), normal(n, outputs, dtype=dtype, seed=3)
    z = x.double() @ w.double().t()
    mass = x.double().abs() @ w.double().abs().t()
    for k, name in enumerate(ACT):
        for bias, residual, keep in ((b, r, True), (None, None, False)) if k else ((b, None, True), (None, r, False)):
            zb = z + (bias.double() if bias is not None else 0.0)
            off = (inputs + 2) * STEP * (mass + zb.abs())
            got = lm.linear(x, w, bias, name, residual, keep_pre=keep)
            if keep:
                near(got[1], zb, off)
                got = got[0]
            want = ACT[name][0](zb) + (residual.double() if residual is not None else 0.0)
            near(got, want, SLOPE * off + EVAL * (zb.abs() + want.abs()))
            if keep:
                assert torch.equal(got, lm.linear(x, w, bias, name, residual))
    # strides that fit no vector access, an output of the caller's, in place of the residual
    out = strided(r, 1)
    wanted = lm.linear(x, w, b, "silu", r)
    assert torch.equal(lm.linear(strided(x, 3), strided(w, 5), b, "silu", out, out=out), wanted)
    assert torch.equal(out, wanted)
    out = strided(r, 8)
    assert torch.equal(lm.linear(strided(x, 8), strided(w, 8), b, "silu", r, out=out), wanted)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,inputs,outputs", LINEAR)
def test_linear_backward(n, inputs, outputs, dtype):
    x, w = normal(n, inputs, dtype=dtype), normal(outputs, inputs, dtype=dtype, scale=inputs ** -0.5, seed=1)
    g, pre, skip = normal(n, outputs, dtype=dtype, seed=2), normal(n, outputs, dtype=dtype, seed=3), normal(n, inputs, dtype=dtype, seed=4)
    half = torch.finfo(dtype).eps / 2
    for name in ACT:
        dz = g.double() * ACT[name][1](pre.double())
        dz_off = half * dz.abs() * 1.01 + EVAL * g.double().abs() * (pre.double().abs() + 1) + (2.0 ** -25 if dtype is torch.float16 else 0)
        for add in (None, skip):
            dx, dw, db = lm.linear_backward(g, x, w, None if name == "identity" else pre, name, skip=add)
            want = dz @ w.double() + (add.double() if add is not None else 0.0)
            near(dx, want, dz_off @ w.double().abs() + (outputs + 2) * STEP * (dz.abs() @ w.double().abs() + want.abs()))
            near(dw, dz.t() @ x.double(), dz_off.t() @ x.double().abs() + (n + 2) * STEP * (dz.abs().t() @ x.double().abs()))
            exact_off = EVAL * g.double().abs() * (pre.double().abs() + 1)
            near(db, dz.sum(0), exact_off.sum(0) + (n + 2) * STEP * dz.abs().sum(0))
        again = lm.linear_backward(strided(g, 3), strided(x, 1), strided(w, 7), strided(pre, 5), name, bias=False, skip=strided(skip, 1))
        assert len(again) == 2 and torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,inputs,outputs", [(2500, 1030, 3000), (300, 4000, 300), (1500, 30000, 1500), (30000, 1500, 1500)])
def test_linear_of_many_tiles(n, inputs, outputs, dtype):
    """Tiles of two blocks, sums cut into parts with either kind of tile, ragged edges of both."""
    x, w = normal(n, inputs, dtype=dtype), normal(outputs, inputs, dtype=dtype, scale=inputs ** -0.5, seed=1)
    b, r = normal(outputs, dtype=dtype, seed=2), normal(n, outputs, dtype=dtype, seed=3)
    z, mass = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t()
    off = (inputs + 2) * STEP * (mass + z.abs())
    got, pre = lm.linear(x, w, b, "gelu", r, keep_pre=True)
    near(pre, z, off)
    want = ACT["gelu"][0](z) + r.double()
    near(got, want, SLOPE * off + EVAL * (z.abs() + want.abs()))
    del z, mass, off, want
    dx, dw, db = lm.linear_backward(r, x, w, pre, "identity", skip=x)
    g = r.double()                      # (no slope: dz is grad itself)
    want = g @ w.double() + x.double()
    near(dx, want, (outputs + 2) * STEP * (g.abs() @ w.double().abs() + want.abs()))
    near(dw, g.t() @ x.double(), (n + 2) * STEP * (g.abs().t() @ x.double().abs()))
    near(db, g.sum(0), (n + 2) * STEP * g.abs().sum(0))
    assert torch.equal(dw, lm.linear_backward(r, x, w)[1])


@pytest.mark.parametrize("dtype", HALVES)
def test_linear_gradient_is_the_slope_of_linear(dtype):
    """Differences of the plain form in 64 bits, along random directions, against the kernels' gradients."""
    n, inputs, outputs = 40, 24, 56
    x, w, b = normal(n, inputs, dtype=dtype), normal(outputs, inputs, dtype=dtype, scale=0.2, seed=1), normal(outputs, dtype=dtype, seed=2)
    g = normal(n, outputs, dtype=dtype, seed=3)
    for name in ("gelu", "silu"):
        pre = lm.linear(x, w, b, name, keep_pre=True)[1]
        dx, dw, db = lm.linear_backward(g, x, w, pre, name)
        value = lambda x, w, b: (g.double() * ACT[name][0](x @ w.t() + b)).sum()
        for k, (at, grad) in enumerate(((x, dx), (w, dw), (b, db))):
            d = normal(*at.shape, seed=7 + k).double()
            args = [[t.double() for t in (x, w, b)] for _ in range(2)]
            h = 1e-4
            args[0][k] = args[0][k] + h * d
            args[1][k] = args[1][k] - h * d
            slope = (value(*args[0]) - value(*args[1])) / (2 * h)
            got = (grad.double() * d).sum()
            # a random direction meets the gradient's roundings (pre, dz, the result) at random signs; all of them
            # at their worst sign stay below 4 half steps of the sum of magnitudes of the terms
            z = x.double() @ w.double().t() + b.double()
            dz = (g.double().abs() * SLOPE)
            mass = ((dz @ w.double().abs()) * d.abs()).sum() if k == 0 else ((dz.t() @ x.double().abs()) * d.abs()).sum() if k == 1 else (dz.sum(0) * d.abs()).sum()
            assert (slope - got).abs() <= 4 * torch.finfo(dtype).eps / 2 * mass * (1 + z.abs().max()) + 1e-6 * mass


def test_no_rows_and_not_numbers():
    x, w, b = normal(0, 16, dtype=torch.bfloat16), normal(40, 16, dtype=torch.bfloat16), normal(40, dtype=torch.bfloat16)
    assert lm.linear(x, w, b).shape == (0, 40)
    dx, dw, db = lm.linear_backward(x.new_empty(0, 40), x, w)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    labels = torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = lm.class_loss(x, w, labels, b)
    assert loss.shape == lse.shape == (0,)
    dx, dw, db = lm.class_loss_backward(loss, x, w, labels, lse, b)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    # a NaN or an infinity stays in its row
    x = normal(200, 16, dtype=torch.bfloat16)
    clean = lm.linear(x, w, b, "relu")
    x[7, 3], x[150, 0] = float("nan"), float("inf")
    got = lm.linear(x, w, b, "identity")
    assert got[7].isnan().all() and not torch.isfinite(got[150]).any()
    rest = [i for i in range(200) if i not in (7, 150)]
    assert torch.equal(lm.linear(x, w, b, "relu")[rest], clean[rest])
    labels = torch.arange(200, device="cuda") % 40
    loss, lse = lm.class_loss(x, w, labels, b)
    assert loss[7].isnan() and torch.isfinite(loss[rest]).all()


def class_case(n, width, classes, dtype, bias=True, seed=0):
    x, w = normal(n, width, dtype=dtype, seed=seed), normal(classes, width, dtype=dtype, scale=2 * width ** -0.5, seed=seed + 1)
    b = normal(classes, dtype=dtype, seed=seed + 2) if bias else None
    g = torch.Generator().manual_seed(seed)
    labels = torch.randint(0, classes, (n,), generator=g).cuda()
    labels[torch.rand(n, generator=g).cuda() < 0.1] = -1
    if n > 2:
        labels[1], labels[2] = classes, classes - 1     # one behind the last class, the last class
    return x, w, b, labels


def plain_loss(x, w, b, labels):
    z = x.double() @ w.double().t() + (b.double() if b is not None else 0.0)
    lse = torch.logsumexp(z, 1)
    live = (labels >= 0) & (labels < w.shape[0])
    at = torch.where(live, labels, 0).long()
    return z, lse, torch.where(live, lse - z.gather(1, at[:, None])[:, 0], 0.0), live, at


CLASSES = [(1, 8, 2), (1, 512, 4000), (3, 5, 1), (4, 17, 7), (31, 64, 26), (64, 33, 64), (65, 96, 65), (128, 128, 256),
           (200, 72, 255), (129, 250, 1030), (300, 16, 5003), (513, 40, 777), (1100, 24, 300), (3000, 136, 5000)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,width,classes", CLASSES)
def test_class_loss_and_its_gradient(n, width, classes, dtype):
    for bias in (True, False):
        x, w, b, labels = class_case(n, width, classes, dtype, bias)
        z, lse, loss, live, at = plain_loss(x, w, b, labels)
        zoff = ((width + 4) * STEP * (x.double().abs() @ w.double().abs().t() + z.abs())).max(1).values
        # the sum of exponentials: at most 256 + tiles additions one behind the other, exponentials off by 4 steps,
        # arguments off by a step of |z| + |max|
        off = zoff + (600 + classes / 64) * STEP + 8 * STEP * (z.abs().max(1).values + 1)
        got, got_lse = lm.class_loss(x, w, labels, b)
        near(got_lse, lse, off)
        near(got, loss, 2 * off)
        assert (got[~live] == 0).all()
        for again in (lm.class_loss(strided(x, 3), strided(w, 1), labels.int(), b), lm.class_loss(strided(x, 8), w, labels, b)):
            assert torch.equal(again[0], got) and torch.equal(again[1], got_lse)

        weights = torch.rand(n, device="cuda") * 2 / n - 0.3 / n
        lse32 = lse.float()
        p = torch.exp(z - lse32.double()[:, None])
        hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
        gl = torch.where(live, weights.double(), 0.0)[:, None]
        dz = gl * (p - hot)
        half = torch.finfo(dtype).eps / 2
        # scores off by zoff, arguments by a step of their size; rounding of dz; below fp16's normal range half of
        # 2^-24 in units of 1 / scale <= 2^-12 of the largest weight
        raw = gl.abs() * p * (zoff[:, None] + 8 * STEP * (z.abs() + lse.abs()[:, None] + 1)) + gl.abs() * STEP
        dz_off = raw + half * dz.abs() * 1.01 + (weights.abs().max().double() * 2.0 ** -37 if dtype is torch.float16 else 0.0)
        outs = lm.class_loss_backward(weights, x, w, labels, lse32, b)
        near(outs[0], dz @ w.double(), dz_off @ w.double().abs() + (classes + 4) * STEP * (dz.abs() @ w.double().abs()))
        near(outs[1], dz.t() @ x.double(), dz_off.t() @ x.double().abs() + (n + 4) * STEP * (dz.abs().t() @ x.double().abs()))
        if bias:
            near(outs[2], dz.sum(0), raw.sum(0) + (n + 4) * STEP * dz.abs().sum(0))
        for again in (lm.class_loss_backward(weights, strided(x, 3), strided(w, 1), labels.int(), lse32, b),
                      lm.class_loss_backward(weights, strided(x, 8), w, labels, lse32, b)):
            assert all(torch.equal(p, q) for p, q in zip(again, outs))


def test_class_loss_in_several_pieces():
    """More scores than a piece of the workspace holds, with the largest type range in the row weights."""
    n, width, classes = 9000, 16, 12000
    x, w, b, labels = class_case(n, width, classes, torch.float16)
    z, lse, loss, live, at = plain_loss(x, w, b, labels)
    weights = torch.rand(n, device="cuda") * 1e-6
    p = torch.exp(z - lse.float().double()[:, None])
    p.scatter_add_(1, at[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
    dz = p.mul_(torch.where(live, weights.double(), 0.0)[:, None])
    outs = lm.class_loss_backward(weights, x, w, labels, lse.float(), b)
    half = torch.finfo(torch.float16).eps / 2
    tiny = weights.max().double() * 2.0 ** -37
    rel = 1.01 * half + 1e-4    # (fp32 scores of 16 terms and their exponentials: below 1e-4)
    a = dz.abs()
    near(outs[0], dz @ w.double(), (a * rel + tiny) @ w.double().abs() + classes * STEP * (a @ w.double().abs()))
    near(outs[1], dz.t() @ x.double(), (a * rel + tiny).t() @ x.double().abs() + n * STEP * (a.t() @ x.double().abs()))
    near(outs[2], dz.sum(0), 1e-4 * a.sum(0) + n * STEP * a.sum(0))


@pytest.mark.parametrize("dtype", HALVES)
def test_forbidden_classes_and_rows_of_them(dtype):
    n, width, classes = 40, 24, 600
    x, w, b, labels = class_case(n, width, classes, dtype)
    b[100:500] = float("-inf")
    b[-1] = torch.finfo(dtype).min
    labels[5] = 200                          # a label that is forbidden
    z, lse, loss, live, at = plain_loss(x, w, b, labels)
    got, got_lse = lm.class_loss(x, w, labels, b)
    assert torch.isfinite(got_lse).all() and got[5] == float("inf")
    near(got_lse, lse, 1e-4)
    near(got, loss, 1e-4 + 2e-6 * loss.abs().nan_to_num(0, 0, 0))
    weights = torch.full((n,), 1.0 / n, device="cuda")
    outs = lm.class_loss_backward(weights, x, w, labels, got_lse, b)
    assert all(torch.isfinite(o).all() for o in outs)
    hot = torch.zeros_like(z).scatter_(1, at[:, None], 1.0)
    dz = torch.where(live, 1.0 / n, 0.0)[:, None].double() * (torch.exp(z - lse[:, None]) - hot)
    rel = torch.finfo(dtype).eps / 2 + 2e-4
    near(outs[1], dz.t() @ x.double(), rel * (dz.abs().t() @ x.double().abs()) + 2e-9)
    # every class forbidden: lse is -inf, a row without a label still has loss 0
    b[:] = float("-inf")
    loss, lse = lm.class_loss(x, w, labels, b)
    assert (lse == float("-inf")).all() and (loss[~live] == 0).all() and loss[live].isnan().all()


def test_streams_graphs_and_workspaces():
    """Each operator on a side stream, and two captured graphs that are replayed by turns with eager calls."""
    forest, _ = grown(40, 5)
    leaves = lm.LeafMap(forest)
    ids = draw_ids(forest, 300)
    dt = torch.bfloat16
    table, x, w, b = normal(leaves.num_rows, 64, dtype=dt), normal(300, 64, dtype=dt), normal(520, 64, dtype=dt), normal(520, dtype=dt)
    g, labels, weights = normal(300, 520, dtype=dt), torch.arange(300, device="cuda"), torch.full((300,), 1 / 300, device="cuda")

    def every(x, stream=None):
        loss, lse = lm.class_loss(x, w, labels, b, stream=stream)
        return [lm.leaf_sum(leaves, ids, table, stream=stream), lm.leaf_sum_backward(leaves, ids, x, stream=stream),
                *lm.linear(x, w, b, "gelu", g, keep_pre=True, stream=stream), *lm.linear_backward(g, x, w, g, "silu", stream=stream),
                loss, lse, *lm.class_loss_backward(weights, x, w, labels, lse, b, stream=stream)]
    want = [every(x), every(x * 2)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for got in (every(x, side),):
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
    with torch.cuda.stream(side):
        got = every(x)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
    graphs, outs, fed = [], [], [x.clone(), x * 2]
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(every(fed[k]))
        graphs.append(graph)
    for turn in range(3):
        for k in (0, 1):
            for o in outs[k]:
                o.zero_()
            graphs[k].replay()
            eager = every(x)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs[k], want[k]))
            assert all(torch.equal(p, q) for p, q in zip(eager, want[0]))


def test_refusals_on_the_device():
    forest, _ = grown(3, 3)
    leaves = lm.LeafMap(forest)
    x, w = normal(8, 16, dtype=torch.bfloat16), normal(16, 16, dtype=torch.bfloat16)
    for call in (lambda: lm.linear(x, w.cpu()), lambda: lm.linear(x, w, out=x), lambda: lm.linear(x, w, residual=normal(8, 16, dtype=torch.bfloat16), out=w[:8]),
                 lambda: lm.leaf_sum(leaves, torch.zeros(2, 3, dtype=torch.int32, device="cuda"), normal(leaves.num_rows, 4).cpu()),
                 lambda: lm.LeafModel(forest, normal(leaves.num_rows, 4), [(w, None, "relu", False)], w)):
        with pytest.raises(kernels.TbkError) as e:
            call()
        assert e.value.status == 1


@pytest.mark.parametrize("dtype", HALVES)
def test_a_model_from_rows_to_gradients(dtype):
    """Forest, leaves, sum, two layers (one residual) and classes in one chain, and the gradients of all parameters
    against differentiation in 64 bits of the same chain without any rounding between."""
    forest, marg = grown(30, 5)
    rows = torch.from_numpy(marg.sample_rows(np.random.default_rng(0), 500)).cuda()
    params = dict(table=normal(lm.LeafMap(forest).num_rows, 48, dtype=dtype, scale=30 ** -0.5), w1=normal(96, 48, dtype=dtype, scale=48 ** -0.5, seed=1),
                  b1=normal(96, dtype=dtype, scale=0.1, seed=2), w2=normal(96, 96, dtype=dtype, scale=96 ** -0.5, seed=3),
                  wc=normal(700, 96, dtype=dtype, scale=96 ** -0.5, seed=4), bc=normal(700, dtype=dtype, scale=0.1, seed=5))
    p = params
    model = lm.LeafModel(forest, p["table"], [(p["w1"], p["b1"], "gelu", False), (p["w2"], None, "silu", True)], p["wc"], p["bc"])
    labels = torch.arange(500, device="cuda") * 13 % 700
    labels[::50] = -1
    loss, grads = model.loss_and_grads(rows, labels)
    assert torch.equal(loss, model.loss(rows, labels))

    q = {k: v.double().requires_grad_(True) for k, v in params.items()}
    at = table_rows(forest, model.forest.predict_leaf_ids(rows))
    h = q["table"][at].sum(1)
    h = ACT["gelu"][0](h @ q["w1"].t() + q["b1"])
    h = ACT["silu"][0](h @ q["w2"].t()) + h
    z = h @ q["wc"].t() + q["bc"]
    live = labels >= 0
    want = torch.where(live, torch.logsumexp(z, 1) - z.gather(1, labels.clamp(min=0)[:, None])[:, 0], 0.0)
    want.mean().backward()
    # each of the six 16-bit roundings on the way is at most eps / 2 of a value; over sums of many terms of random
    # sign they add up as their squares, to about sqrt(6) eps / 2 of the result in the 2-norm: 8 eps / 2 covers it
    half = torch.finfo(dtype).eps / 2
    assert (loss.double() - want).norm() <= 8 * half * want.norm()
    got = dict(table=grads["table"], w1=grads["layers"][0][0], b1=grads["layers"][0][1], w2=grads["layers"][1][0], wc=grads["weight"], bc=grads["bias"])
    assert grads["layers"][1][1] is None
    for k in q:
        assert (got[k].double() - q[k].grad).norm() <= 8 * half * q[k].grad.norm(), k
    scores = model.scores(rows[:1])
    assert scores.shape == (1, 700) and (scores.double() - z[:1].detach()).norm() <= 8 * half * z[:1].norm()


def complete_forest(trees, levels):
    """Complete trees as flat arrays, leaves last; the row of leaf i of tree t is t << levels | i."""
    from types import SimpleNamespace
    inner, nodes = (1 << levels) - 1, (2 << levels) - 1
    at = np.arange(nodes)
    return SimpleNamespace(num_trees=trees, tree_off=np.arange(trees + 1, dtype=np.int64) * nodes,
                           left=np.tile(np.where(at < inner, 2 * at + 1, -1).astype(np.int32), trees),
                           right=np.tile(np.where(at < inner, 2 * at + 2, -1).astype(np.int32), trees),
                           feat=np.zeros(trees * nodes, np.int32), thr=np.zeros(trees * nodes, np.float32),
                           class_id=np.zeros(trees, np.int32), num_classes=0, transform=0, initial_value=0.0, num_features=1)


@pytest.mark.parametrize("dtype,trees,levels,n,width", [
    (torch.bfloat16, 37, 6, 10001, 64), (torch.float16, 100, 8, 19999, 64), (torch.bfloat16, 20, 7, 12345, 120),
    (torch.float32, 21, 5, 11111, 100), (torch.float16, 5, 4, 160001, 256), (torch.bfloat16, 9, 9, 20000, 64)])
def test_leaf_sum_of_many_rows(dtype, trees, levels, n, width):
    """Tables in shared memory (and, in the last case, too large for it), ragged tiles and batches of trees, struck-out
    ids, ids at odd addresses, tables that do not lie row behind row."""
    forest = complete_forest(trees, levels)
    leaves = lm.LeafMap(forest)
    g = torch.Generator(device="cuda")
    g.manual_seed(trees)
    leaf = (torch.rand(n, trees, generator=g, device="cuda") ** 2 * (1 << levels)).int()
    ids = leaf + (1 << levels) - 1
    gone = torch.rand(n, trees, generator=g, device="cuda") < 0.05
    ids[gone] = torch.randint(-3, (1 << levels) - 1, (int(gone.sum()),), generator=g, device="cuda", dtype=torch.int32)
    table = normal(leaves.num_rows, width, dtype=dtype)
    want, mass = torch.zeros(n, width, dtype=torch.float64, device="cuda"), torch.zeros(n, width, dtype=torch.float64, device="cuda")
    for t in range(trees):
        rows = table.double()[(t << levels) + leaf[:, t].long()] * ~gone[:, t, None]
        want += rows
        mass += rows.abs()
    near(lm.leaf_sum(leaves, ids, table), want, trees * STEP * mass)
    odd = torch.full((n, trees + 3), -1, dtype=torch.int32, device="cuda")
    odd[:, 1:trees + 1] = ids
    assert torch.equal(lm.leaf_sum(leaves, odd[:, 1:trees + 1], table), lm.leaf_sum(leaves, ids, table))
    near(lm.leaf_sum(leaves, ids, strided(table, 8)), want, trees * STEP * mass)
    near(lm.leaf_sum(leaves, ids, strided(table, 1)), want, trees * STEP * mass)


def test_leaf_gradient_of_trees_beyond_two_byte_leaf_numbers():
    forest = complete_forest(2, 17)
    leaves = lm.LeafMap(forest)
    leaf = torch.randint(0, 1 << 17, (5000, 2), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    leaf[::3] = (1 << 17) - 1
    grad = normal(5000, 8)
    rows = leaf + torch.tensor([0, 1 << 17], device="cuda")
    want = torch.zeros(leaves.num_rows, 8, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want)
    for t in range(2):
        want.index_add_(0, rows[:, t], grad.double())
        mass.index_add_(0, rows[:, t], grad.double().abs())
    near(lm.leaf_sum_backward(leaves, (leaf + (1 << 17) - 1).int(), grad), want, 5000 * STEP * mass)


@pytest.mark.parametrize("n", [3, 700])
def test_leaf_sum_past_four_gigabytes_of_table(n):
    trees, levels, width = 70, 16, 512
    leaves = lm.LeafMap(complete_forest(trees, levels))
    table = torch.empty(leaves.num_rows, width, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    assert table.numel() > 1 << 31
    leaf = torch.randint(0, 1 << levels, (n, trees), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    rows = leaf + (torch.arange(trees, device="cuda") << levels)
    picked = table[rows.reshape(-1)].view(n, trees, width).double()
    near(lm.leaf_sum(leaves, (leaf + (1 << levels) - 1).int(), table), picked.sum(1), trees * STEP * picked.abs().sum(1))


@pytest.mark.parametrize("outputs", [4100, 4104])
def test_linear_past_two_gigaelements(outputs):
    n, inputs = 530000, 24
    assert n * outputs > 1 << 31
    x, w = normal(n, inputs, dtype=torch.bfloat16), normal(outputs, inputs, dtype=torch.bfloat16, seed=1)
    got = lm.linear(x, w)
    for a in (0, 523000, n - 300):
        z, mass = x[a:a + 300].double() @ w.double().t(), x[a:a + 300].double().abs() @ w.double().abs().t()
        near(got[a:a + 300], z, (inputs + 2) * STEP * mass)


@pytest.mark.parametrize("n", [7, 8, 9, 16])
def test_linear_around_few_rows(n):
    for inputs, outputs in ((100, 70), (1032, 515), (8, 9), (2056, 1000)):
        x, w, b, r = (normal(*s, dtype=torch.float16, seed=i) for i, s in enumerate(((n, inputs), (outputs, inputs), (outputs,), (n, outputs))))
        z, mass = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t()
        off = (inputs + 2) * STEP * (mass + z.abs())
        got, pre = lm.linear(x, w, b, "silu", r, keep_pre=True)
        near(pre, z, off)
        want = ACT["silu"][0](z) + r.double()
        near(got, want, SLOPE * off + EVAL * (z.abs() + want.abs()))


def test_calls_of_two_streams_at_once():
    forest, _ = grown(60, 6)
    leaves = lm.LeafMap(forest)
    ids = draw_ids(forest, 12000)
    table = normal(leaves.num_rows, 64, dtype=torch.bfloat16)
    x, w = normal(3000, 200, dtype=torch.bfloat16), normal(5000, 200, dtype=torch.bfloat16)
    labels, weights = torch.arange(3000, device="cuda"), torch.full((3000,), 1 / 3000, device="cuda")

    def work():
        loss, lse = lm.class_loss(x, w, labels)
        return [lm.leaf_sum(leaves, ids, table), lm.leaf_sum_backward(leaves, ids, lm.leaf_sum(leaves, ids, table)), loss,
                *lm.class_loss_backward(weights, x, w, labels, lse), *lm.linear_backward(x, x, w[:200], None, "identity")]
    want = work()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(work())
    torch.cuda.synchronize()
    for outs in got[0] + got[1]:
        assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_extreme_values_of_activations():
    """Far tails, zeros of both signs and infinities, as the formulas have them."""
    z = torch.tensor([-60000.0, -100.0, -20.0, -6.0, -5e-8, -0.0, 0.0, 5e-8, 6.0, 20.0, 100.0, 60000.0, float("inf")], device="cuda").half()
    x, one = z[:, None].contiguous(), torch.ones(1, 1, dtype=torch.float16, device="cuda")
    wide = torch.ones(40, 1, dtype=torch.float16, device="cuda")
    for name in ("relu", "gelu", "silu"):
        want = ACT[name][0](z.double())
        for got in (lm.linear(x, one, activation=name)[:, 0], lm.linear(x[:5], one, activation=name)[:, 0], lm.linear(x, wide, activation=name)[:, 33]):
            near(got, want[:len(got)], EVAL * z[:len(got)].double().abs().clamp(max=1e5))
        dz = lm.linear_backward(torch.ones_like(x[:-1]), x[:-1], one, x[:-1], name)[0][:, 0]
        near(dz, ACT[name][1](z[:-1].double()), EVAL * (z[:-1].double().abs().clamp(max=100) + 1) + 2.0 ** -11)


def test_a_graph_that_forks_and_joins():
    """Calls behind waits for another stream's events, inside one captured graph."""
    forest, _ = grown(20, 5)
    leaves = lm.LeafMap(forest)
    ids = draw_ids(forest, 500)
    table, w = normal(leaves.num_rows, 64, dtype=torch.bfloat16), normal(300, 64, dtype=torch.bfloat16)
    labels = torch.arange(500, device="cuda") % 300

    def forked(side):
        h = lm.leaf_sum(leaves, ids, table)
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            y = lm.linear(h, w, activation="gelu")
        loss, lse = lm.class_loss(h, w, labels)
        here.wait_stream(side)
        dx, dw = lm.linear_backward(y, h, w, y, "silu", bias=False)
        return [h, y, loss, lse, dx, dw, lm.leaf_sum_backward(leaves, ids, dx)]
    side = torch.cuda.Stream()
    want = forked(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = forked(side)
    for _ in range(3):
        for o in got:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_small_and_large_weights_of_rows():
    """Row weights far outside fp16's range, rows of weight zero among them, and one that is not finite."""
    for dtype in HALVES:
        for size in (1e-30, 1e-9, 1.0, 1e6):
            x, w, b, labels = class_case(300, 48, 500, dtype)
            z, lse, _, live, at = plain_loss(x, w, b, labels)
            weights = torch.rand(300, device="cuda") * size
            weights[::7] = 0
            p = torch.exp(z - lse.float().double()[:, None])
            p.scatter_add_(1, at[:, None], torch.full((300, 1), -1.0, dtype=torch.float64, device="cuda"))
            dz = p * torch.where(live, weights.double(), 0.0)[:, None]
            outs = lm.class_loss_backward(weights, x, w, labels, lse.float(), b)
            rel, tiny = 1.01 * torch.finfo(dtype).eps / 2 + 1e-4, weights.max().double() * 2.0 ** -37
            # results below the type's own range round to its grid: half a step of its smallest subnormal number
            grid = 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -134
            mass = dz.abs() * rel + tiny
            near(outs[1], dz.t() @ x.double(), mass.t() @ x.double().abs() + 300 * STEP * (dz.abs().t() @ x.double().abs()) + grid)
            near(outs[2], dz.sum(0), 1e-4 * dz.abs().sum(0) + 300 * STEP * dz.abs().sum(0) + grid)
    # (the last weights are beyond fp16's range themselves: the other rows stay what they were, infinities among them)
    before, rest = outs[0], [i for i in range(300) if i != 5]
    weights[5], labels[5] = float("inf"), 3
    outs = lm.class_loss_backward(weights, x, w, labels, lse.float(), b)
    assert torch.equal(outs[0][rest], before[rest]) and not torch.isfinite(outs[0][5]).any()


def test_a_closed_map_is_not_read():
    forest, _ = grown(3, 3)
    leaves = lm.LeafMap(forest)
    ids, rows = draw_ids(forest, 5), leaves.num_rows
    lm.leaf_sum(leaves, ids, normal(rows, 8))
    leaves.close()
    for call in (lambda: lm.leaf_sum(leaves, ids, normal(rows, 8)), lambda: lm.leaf_sum_backward(leaves, ids, normal(5, 8))):
        with pytest.raises(kernels.TbkError) as e:
            call()
        assert e.value.status == 1


@pytest.mark.parametrize("n", [0, 1])
def test_a_model_of_few_or_no_rows(n):
    forest, marg = grown(4, 3)
    params = [normal(int((np.asarray(forest.left) < 0).sum()), 16, dtype=torch.bfloat16), normal(16, 16, dtype=torch.bfloat16, seed=1), normal(9, 16, dtype=torch.bfloat16)]
    model = lm.LeafModel(forest, params[0], [(params[1], None, "silu", True)], params[2])
    rows = torch.from_numpy(marg.sample_rows(np.random.default_rng(0), 2))[:n].cuda()
    loss, grads = model.loss_and_grads(rows, torch.zeros(n, dtype=torch.int64, device="cuda"))
    assert loss.shape == (n,) and model.scores(rows).shape == (n, 9)
    for got, like in ((grads["table"], params[0]), (grads["layers"][0][0], params[1]), (grads["weight"], params[2])):
        assert got.shape == like.shape and torch.isfinite(got).all() and bool((got != 0).any()) == (n > 0)
