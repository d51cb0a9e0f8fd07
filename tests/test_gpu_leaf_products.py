"""Launches that carry both products of a backward pass, at sizes where blocks pass from one to the other and the two
leave their results in different ways (by find_cut on 148 multiprocessors; the comments say how).

Tolerances as in test_gpu_leaf_model.py."""
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_leaf_model import HALVES, STEP, class_case, near, no_wait_gave_up, normal, plain_loss  # noqa: F401
from treebeard_b200 import leaf_model as lm

pytestmark = pytest.mark.gpu


def class_gradients_are_near(outs, x, w, b, labels, weights, z, lse, live, at):
    """lse: what the call was given.  Errors of dz: scores off by their sums' steps, arguments of the exponentials by a
    step of their size, the rounding to 16 bits, and below fp16's normal range half of 2^-24 in units of
    1 / scale <= 2^-12 of the largest weight of a row with a label."""
    (n, width), classes = x.shape, w.shape[0]
    X, W, dtype = x.double(), w.double(), x.dtype
    p = torch.exp(z - lse.double()[:, None])
    gl = torch.where(live, weights.double(), 0.0)[:, None]
    zoff = (width + 4) * STEP * (X.abs() @ W.abs().t() + z.abs())
    raw = gl.abs() * (p * (zoff + 8 * STEP * (z.abs() + lse.double().abs()[:, None] + 1)) + STEP)
    del zoff
    dz = gl * p.scatter_add_(1, at[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
    tiny = gl.abs().max() * 2.0 ** -37 if dtype is torch.float16 else 0.0
    off = raw + torch.finfo(dtype).eps / 2 * dz.abs() * 1.01 + tiny
    near(outs[0], dz @ W, off @ W.abs() + (classes + 4) * STEP * (dz.abs() @ W.abs()))
    near(outs[1], dz.t() @ X, off.t() @ X.abs() + (n + 4) * STEP * (dz.abs().t() @ X.abs()))
    if b is not None:
        near(outs[2], dz.sum(0), raw.sum(0) + (n + 4) * STEP * dz.abs().sum(0))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,width,classes", [
    (128, 64, 32768),     # 128 x 128: 32 parts of x's gradient, then whole tiles of the weights'
    (1024, 512, 32000),   # 256 x 256: 8 parts, then whole tiles
    (200, 600, 20000),    # 256 x 256: 16 parts, then whole tiles, ragged
    (2048, 2048, 50257),  # 512 x 256: 2 parts, then whole tiles
])
def test_class_gradient_of_parts_and_whole_sums(n, width, classes, dtype):
    x, w, b, labels = class_case(n, width, classes, dtype)
    z, lse, _, live, at = plain_loss(x, w, b, labels)
    weights = (torch.rand(n, device="cuda") + 0.5) / n
    lse = lse.float()
    outs = lm.class_loss_backward(weights, x, w, labels, lse, b)
    for _ in range(20):    # (nothing that depends on which copy ends when)
        assert all(torch.equal(p, q) for p, q in zip(outs, lm.class_loss_backward(weights, x, w, labels, lse, b)))
    class_gradients_are_near(outs, x, w, b, labels, weights, z, lse, live, at)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n,inputs,outputs", [
    (100, 37900, 100),    # 128 x 128: each block has two tiles with skip, then two of the weights'
    (60, 40000, 120),
    (801, 3823, 33),      # one tile with skip, then one of the weights'
    (132, 2414, 1907),    # 256 x 256: five parts, then whole tiles
    (6189, 598, 33),      # whole tiles with skip, then twenty parts
    (272, 3577, 1760),    # whole tiles of either
])
def test_layer_gradient_with_skip_and_the_weights_in_one_launch(n, inputs, outputs, dtype):
    x, w = normal(n, inputs, dtype=dtype), normal(outputs, inputs, dtype=dtype, scale=inputs ** -0.5, seed=1)
    g, skip = normal(n, outputs, dtype=dtype, seed=2), normal(n, inputs, dtype=dtype, seed=4)
    G, X, W = g.double(), x.double(), w.double()
    for add in (skip, None):
        outs = lm.linear_backward(g, x, w, skip=add)
        for _ in range(20):
            assert all(torch.equal(p, q) for p, q in zip(outs, lm.linear_backward(g, x, w, skip=add)))
        want = G @ W + (add.double() if add is not None else 0.0)
        near(outs[0], want, (outputs + 2) * STEP * (G.abs() @ W.abs() + want.abs()))
        near(outs[1], G.t() @ X, (n + 2) * STEP * (G.abs().t() @ X.abs()))
        near(outs[2], G.sum(0), (n + 2) * STEP * G.abs().sum(0))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [0.0, 1e6, 1e9, 1e30, float("inf"), float("nan")])
def test_weights_of_rows_without_a_label_do_not_count(size, dtype):
    """Rows without a label have zeros for dz: their weights change no bit of the gradients."""
    n, width, classes = 300, 64, 1000
    x, w, b, labels = class_case(n, width, classes, dtype)
    z, lse, _, live, at = plain_loss(x, w, b, labels)
    assert 3 < int((~live).sum()) < n // 2
    weights = torch.full((n,), 1.0 / n, device="cuda")
    outs = []
    for kind in (torch.int64, torch.int32):
        given = torch.where(live, weights, size)
        outs.append(lm.class_loss_backward(given, x, w, labels.to(kind), lse.float(), b))
        assert all(torch.equal(p, q) for p, q in zip(outs[-1], lm.class_loss_backward(weights, x, w, labels, lse.float(), b)))
    class_gradients_are_near(outs[0], x, w, b, labels, weights, z, lse.float(), live, at)
    # no row with a label: zeros everywhere
    for o in lm.class_loss_backward(given, x, w, torch.full_like(labels, -100), lse.float(), b):
        assert (o == 0).all()


def test_the_status_waits_for_every_stream():
    """Streams of torch do not wait for the legacy stream, nor it for them."""
    x, w = normal(256, 256, dtype=torch.bfloat16), normal(256, 256, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    lm.linear(x, w, stream=side)           # (kernels are loaded, memory is there: neither waits below)
    torch.cuda._sleep(1000)
    lm.check_status(0)
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)     # about a tenth of a second
        lm.linear(x, w)
        after = torch.cuda.Event()
        after.record()
    lm.check_status(0)
    assert after.query()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("classes", [1, 2, 31, 300, 1500])
def test_losses_of_sure_rows(classes, bias, dtype):
    """Scores up to 300 that no sum rounds (small whole numbers): a loss is off only by its own exponentials and
    logarithm, however large the scores are, and never below 0; with one class it is 0, and so are all gradients."""
    n = 200
    g = torch.Generator().manual_seed(classes)
    x = torch.randint(-6, 7, (n, 8), generator=g).to(dtype).cuda()
    w = torch.randint(-6, 7, (classes, 8), generator=g).to(dtype).cuda()
    b = torch.randint(-12, 13, (classes,), generator=g).to(dtype).cuda() if bias else None
    z = x.double() @ w.double().t() + (b.double() if bias else 0.0)
    labels = z.argmax(1)                      # (the sure ones; every third row something else)
    labels[::3] = torch.arange(n, device="cuda")[::3] % classes
    loss, lse = lm.class_loss(x, w, labels, b)
    top = z.max(1, keepdim=True).values
    rest = torch.exp(z - top).sum(1).log()
    want = (top - z.gather(1, labels[:, None]))[:, 0] + rest
    # a sum of exponentials relative to the largest: each is off by 2^-22 and, e^-d d <= 0.37, by the roundings of its
    # argument d; 32 additions one behind the other in a chunk and one for each chunk and part: (8 + 16 + classes / 32) steps
    off = (24 + classes / 32) * STEP
    assert (loss >= 0).all() and z.abs().max() > 50
    near(loss, want, off + STEP * want)
    near(lse, top[:, 0] + rest, off + STEP * z.abs().max())
    outs = lm.class_loss_backward(torch.full((n,), 1 / n, device="cuda"), x, w, labels, lse, b)
    if classes == 1:
        assert (loss == 0).all() and torch.equal(lse.double(), z[:, 0]) and all((o == 0).all() for o in outs)


@pytest.mark.parametrize("classes", [5, 300, 3000])
def test_infinite_scores(classes):
    """A row with an infinite score has an infinite logarithm, and so has its loss unless the label is that class."""
    n = 70
    x, w, b, labels = class_case(n, 16, classes, torch.bfloat16)
    b[-1] = float("inf")
    x[3, 0] = float("nan")
    z, lse, loss, live, at = plain_loss(x, w, b, labels)
    got, got_lse = lm.class_loss(x, w, labels, b)
    rest = [i for i in range(n) if i != 3]
    assert (got_lse[rest] == float("inf")).all() and got_lse[3].isnan()
    hit = live & (labels == classes - 1)
    assert hit.any() and got[hit].isnan().all() and (got[~live] == 0).all()
    other = live & ~hit
    other[3] = False
    assert (got[other] == float("inf")).all()


@pytest.mark.parametrize("name", ["relu", "gelu", "silu"])
def test_slopes_where_the_kept_value_rounded_to_infinity(name):
    """In fp16 a value below -65520 is kept as -inf; its slope is 0 and those above 65520 have 1.  NaN stays NaN."""
    x = torch.tensor([[-300.0], [300.0], [2.0], [float("nan")]], device="cuda").half()
    w = torch.tensor([[400.0], [1.0]], device="cuda").half()
    y, pre = lm.linear(x, w, None, name, keep_pre=True)
    assert pre[0, 0] == float("-inf") and pre[1, 0] == float("inf") and y[0, 0] == 0
    g = torch.full((4, 2), 0.5, device="cuda").half()
    dx, dw, db = lm.linear_backward(g[:3], x[:3], w, pre[:3], name)
    assert torch.isfinite(dw).all() and torch.isfinite(db).all()
    slopes = torch.tensor([0.0, 1.0], device="cuda").half()
    assert torch.equal(lm.linear_backward(g[:2, :1], x[:2], torch.ones_like(w[:1]), pre[:2, :1], name)[0][:, 0], 0.5 * slopes)
    if name != "relu":
        assert lm.linear_backward(g[3:], x[3:], w, pre[3:], name)[0].isnan().all()


def test_arguments_that_are_given_up_while_another_stream_reads_them():
    """A temporary's memory is not handed out again before the call on the other stream has read it."""
    w = normal(512, 512, dtype=torch.bfloat16)
    x = normal(2048, 512, dtype=torch.bfloat16)
    want = lm.linear(x * 2, w)
    side = torch.cuda.Stream()
    lm.linear(x, w, stream=side)          # (kernels are loaded, memory is there)
    torch.cuda.synchronize()
    for _ in range(3):
        here = x * 2
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)
        got = lm.linear(here, w, stream=side)
        del here
        foreign = [torch.full_like(x, float("nan")) for _ in range(4)]   # on the current stream, meanwhile
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del foreign


def test_a_captured_call_on_a_forked_stream_with_a_temporary():
    w = normal(512, 512, dtype=torch.bfloat16)
    x = normal(2048, 512, dtype=torch.bfloat16)
    want = lm.linear(x * 2, w)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    lm.linear(x, w, stream=side)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        twice = x * 2
        side.wait_stream(here)
        got = lm.linear(twice, w, stream=side)
        del twice
        foreign = [torch.full_like(x, float("nan")) for _ in range(4)]
        here.wait_stream(side)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and all(f.isnan().all() for f in foreign)
