"""The token operators and AdamW over many tensors on the GPU, against the
plain 64-bit forms of tests/_tokens.py (the 8-bit moments against a
step-by-step f32 form, bit for bit)."""
import ctypes

import numpy as np
import pytest

from rusttorch_b200 import _native as N
from tests import _tokens as K

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]


@pytest.fixture(scope="module")
def rt():
    import rusttorch_b200 as rt
    return rt


def put(rt, a, dtype="float32"):
    a = np.ascontiguousarray(a, np.float32)
    return rt.Tensor.from_numpy(a.astype(np.float16), dtype=None) if dtype == "float16" else rt.Tensor.from_numpy(a, dtype="bfloat16" if dtype == "bfloat16" else None)


def get(t):
    return t.to_numpy().astype(np.float32) if t.dtype == "float16" else t.to_numpy()


def shifted(rt, a, dtype, elements, keep=[]):
    """The same values `elements` elements into a larger buffer (rows that do not start on 16 bytes)."""
    a = np.ascontiguousarray(a, np.float32)
    big = put(rt, np.concatenate([np.full(elements, 9.0, np.float32), a.ravel(), np.full(8, 9.0, np.float32)]), dtype)
    size = N.DTYPE_BYTES[big._code]
    return rt.Tensor.from_device_ptr(big.ptr + elements * size, a.shape, owner=big, dtype=dtype), big


def same(got, want):
    got, want = np.asarray(got, np.float32), np.asarray(want, np.float32)
    assert got.shape == want.shape
    off = (got.view(np.uint32) != want.view(np.uint32)) & ~(np.isnan(got) & np.isnan(want))
    assert not off.any(), (int(off.sum()), np.argwhere(off)[:3].tolist(), got[off][:3], want[off][:3])


def near(got, want, bound):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert (np.isnan(got) == np.isnan(want)).all()
    assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all()
    off = np.abs(got[fine] - want[fine])
    allowed = np.broadcast_to(bound, want.shape)[fine]
    assert np.isfinite(allowed).all()
    worst = int(np.argmax(off - allowed)) if off.size else 0
    assert off.size == 0 or off[worst] <= allowed[worst], (off[worst], allowed[worst], worst)


def no_flag():
    N.check(N.lib().rtc_synchronize())


def flagged():
    with pytest.raises(N.RusttorchError) as e:
        N.check(N.lib().rtc_synchronize())
    assert e.value.code == N.INVALID_ARGUMENT and "outside the vocabulary" in str(e.value)
    no_flag()


# ---- softmax cross entropy ---------------------------------------------------------

def logits_of(n, v, seed, dtype, masked=True):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 3, (n, v)).astype(np.float32)
    t = rng.integers(0, v, n)
    for i in range(n):
        x[i, t[i]] += (14.0, 5.0, 0.0)[i % 3]
    if masked and v > 4:
        x[:, rng.integers(0, v, max(1, v // 50))] = -np.inf
        x[np.arange(n), t] = np.maximum(x[np.arange(n), t], -3)
    if n > 2:
        t[1::7] = -100
    return K.rounded(x, dtype), t


# the longest path of additions that a kernel may take over a row: a thread's own
# elements one after the other in two sums (128 threads at least to a row, or 32
# to one of 400 vectors, 3200 elements, at most), then 10 halvings of a block and
# 4 of a cluster
def chain(v):
    return v // (64 if v <= 3200 else 128) + 16


SHAPES = [(1, 1), (1, 2), (2, 3), (3, 7), (5, 8), (4, 31), (9, 129), (5, 1000), (33, 1024), (300, 257), (6, 4097), (4, 32768), (3, 50257),
          (2, 100003), (3, 131072), (2, 262147), (2, 600001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, v", SHAPES)
def test_loss_forward_backward_and_fused(rt, n, v, dtype):
    x, t = logits_of(n, v, n + v, dtype)
    ids = t.astype(np.int64 if v % 2 else np.int32)
    want, wg = K.token_loss(x, t)
    lb, gb = K.token_loss_bounds(x, t, -100, "mean", 1.0, chain(v), dtype)
    X, T = put(rt, x, dtype), rt.Tensor.from_numpy(ids)
    loss, stats = rt.softmax_cross_entropy(X, T)
    near(loss.to_numpy(), want, lb)
    one = rt.Tensor.from_numpy(np.float32([1.0]))
    near(get(rt.softmax_cross_entropy_backward(one, X, T, stats)), wg, gb)
    loss, grad = rt.softmax_cross_entropy_grad(X, T)
    near(loss.to_numpy(), want, lb)
    near(get(grad), wg, gb)
    # in place: the gradient takes the logits' memory
    rt.softmax_cross_entropy_backward(one, X, T, stats, out=X)
    near(get(X), wg, gb)
    X = put(rt, x, dtype)
    loss, _ = rt.softmax_cross_entropy_grad(X, T, grad=X)
    near(loss.to_numpy(), want, lb)
    near(get(X), wg, gb)
    no_flag()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_loss_reductions_and_scales(rt, reduction, dtype):
    n, v, scale = 37, 513, 2.5
    x, t = logits_of(n, v, 5, dtype)
    want, wg = K.token_loss(x, t, reduction=reduction, scale=scale)
    lb, gb = K.token_loss_bounds(x, t, -100, reduction, scale, chain(v), dtype)
    X, T = put(rt, x, dtype), rt.Tensor.from_numpy(t)
    loss, grad = rt.softmax_cross_entropy_grad(X, T, reduction=reduction, grad_scale=scale)
    near(loss.to_numpy(), want, lb)
    near(get(grad), wg, gb)
    loss, stats = rt.softmax_cross_entropy(X, T, reduction=reduction)
    near(loss.to_numpy(), want, lb)
    up = np.float32(scale) * np.ones(n if reduction == "none" else 1, np.float32)
    near(get(rt.softmax_cross_entropy_backward(rt.Tensor.from_numpy(up), X, T, stats, reduction=reduction)), wg, gb)


def test_loss_rows_have_their_own_upstream(rt):
    n, v = 19, 300
    x, t = logits_of(n, v, 8, "float32")
    up = np.linspace(-2, 2, n).astype(np.float32)
    up[3] = 0.0
    wg = K.token_loss(x, t, reduction="none")[1] * up[:, None].astype(np.float64)
    gb = K.token_loss_bounds(x, t, -100, "none", 1.0, chain(v), "float32")[1] * np.abs(up[:, None]) + 2.0 ** -140
    X, T = put(rt, x), rt.Tensor.from_numpy(t)
    _, stats = rt.softmax_cross_entropy(X, T, reduction="none")
    near(rt.softmax_cross_entropy_backward(rt.Tensor.from_numpy(up), X, T, stats, reduction="none").to_numpy(), wg, gb)


def test_loss_of_many_dimensions(rt):
    x, t = logits_of(12, 50, 2, "float32")
    want, wg = K.token_loss(x, t, reduction="none")
    lb, gb = K.token_loss_bounds(x, t, -100, "none", 1.0, chain(50), "float32")
    X, T = rt.Tensor.from_numpy(x.reshape(3, 4, 50)), rt.Tensor.from_numpy(t.reshape(3, 4))
    loss, grad = rt.softmax_cross_entropy_grad(X, T, reduction="none")
    assert loss.shape() == [3, 4] and grad.shape() == [3, 4, 50]
    near(loss.to_numpy().reshape(-1), want, lb)
    near(grad.to_numpy().reshape(12, 50), wg, gb)
    # one row: logits [V], targets []
    loss, grad = rt.softmax_cross_entropy_grad(rt.Tensor.from_numpy(x[0].copy()), rt.Tensor.from_numpy(np.int64(t[0])), reduction="none")
    near(loss.to_numpy(), want[0], lb[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [40, 9000, 40007, 300001])
def test_loss_of_extreme_rows(rt, v, dtype):
    big = {"float32": 3.4e38, "bfloat16": 3.38e38, "float16": 65504.0}[dtype]
    x = np.zeros((9, v), np.float32)
    t = np.arange(9)
    x[0] = -big                                   # uniform: log V, not 0
    x[1] = -np.inf                                # nothing is left
    x[2, 5] = np.nan
    x[3, 6] = np.inf
    x[4, :] = -np.inf
    x[4, 4] = 1.0                                 # one class left, the target: loss 0
    x[5, 5] = -np.inf                             # the target is ruled out: loss inf, gradient -1
    x[6] = -big
    x[6, 7] = big                                 # differences that overflow: loss inf
    x[7, 7] = 30.0                                # sure: the loss keeps its digits
    x[8, 8] = -30.0
    x = K.rounded(x, dtype)
    X, T = put(rt, x, dtype), rt.Tensor.from_numpy(t)
    want, wg = K.token_loss(x, t, reduction="none")
    with np.errstate(over="ignore"):
        want[6] = np.inf if dtype != "float16" else want[6]
    lb, gb = K.token_loss_bounds(x, t, -100, "none", 1.0, chain(v), dtype)
    for form in ("tape", "fused"):
        if form == "tape":
            loss, stats = rt.softmax_cross_entropy(X, T, reduction="none")
            grad = rt.softmax_cross_entropy_backward(rt.Tensor.from_numpy(np.ones(9, np.float32)), X, T, stats, reduction="none")
        else:
            loss, grad = rt.softmax_cross_entropy_grad(X, T, reduction="none")
        near(loss.to_numpy(), want, lb)
        near(get(grad), wg, gb)
    assert abs(float(loss.to_numpy()[7]) / ((v - 1) * np.exp(-30.0)) - 1) < 1e-3 or dtype != "float32"
    no_flag()


@pytest.mark.parametrize("v", [64, 70000])
def test_loss_of_ignored_and_bad_targets(rt, v):
    x, _ = logits_of(6, v, 4, "float32", masked=False)
    # every row ignored: loss and gradient 0, whatever the logits hold
    x[2, 3] = np.nan
    X = rt.Tensor.from_numpy(x)
    loss, grad = rt.softmax_cross_entropy_grad(X, rt.Tensor.from_numpy(np.full(6, -1)), ignore_index=-1)
    assert float(loss.to_numpy().reshape(())) == 0.0 and (grad.to_numpy() == 0).all()
    loss, stats = rt.softmax_cross_entropy(X, rt.Tensor.from_numpy(np.full(6, -1)), ignore_index=-1)
    grad = rt.softmax_cross_entropy_backward(loss, X, rt.Tensor.from_numpy(np.full(6, -1)), stats, ignore_index=-1)
    assert float(loss.to_numpy().reshape(())) == 0.0 and (grad.to_numpy() == 0).all()
    no_flag()
    # ignore_index inside the vocabulary
    t = np.array([0, 1, 2, 2, 4, 5])
    want, wg = K.token_loss(x, t, ignore=2)
    lb, gb = K.token_loss_bounds(x, t, 2, "mean", 1.0, chain(v), "float32")
    loss, grad = rt.softmax_cross_entropy_grad(X, rt.Tensor.from_numpy(t), ignore_index=2)
    near(loss.to_numpy(), want, lb)
    near(grad.to_numpy(), wg, gb)
    no_flag()
    # targets outside: NaN rows, the others as they are, and a report
    x[2, 3] = 0.0
    X = rt.Tensor.from_numpy(x)
    for bad in (v, -1, 1 << 40, -(1 << 50)):
        t = np.array([0, bad, 2, 3, 4, 5], np.int64)
        want, wg = K.token_loss(x, t, reduction="none")
        lb, gb = K.token_loss_bounds(x, t, -100, "none", 1.0, chain(v), "float32")
        T = rt.Tensor.from_numpy(t)
        loss, grad = rt.softmax_cross_entropy_grad(X, T, reduction="none")
        assert np.isnan(want[1])
        near(loss.to_numpy(), want, lb)
        near(grad.to_numpy(), wg, gb)
        flagged()
        loss, stats = rt.softmax_cross_entropy(X, T, reduction="none")
        flagged()
        grad = rt.softmax_cross_entropy_backward(rt.Tensor.from_numpy(np.ones(6, np.float32)), X, T, stats, reduction="none")
        near(grad.to_numpy(), wg, gb)
        flagged()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [4099, 20001, 70001])
def test_loss_of_many_rows_of_all_kinds(rt, v, dtype):
    """Rows for all SMs, extreme ones, ignored ones and bad targets among them."""
    n = 310
    x, t = logits_of(n, v, 3, dtype)
    big = {"float32": 3.4e38, "bfloat16": 3.38e38, "float16": 65504.0}[dtype]
    x[2] = -big
    x[12] = -np.inf
    x[22, v - 1] = np.nan
    x[32, 0] = np.inf
    x[42] = -np.inf
    x[42, t[42]] = 2.0
    x[52, :] = -big
    x[52, v // 2] = big / 4
    x[62] *= 2.0 ** 20 if dtype != "float16" else 64
    t[72] = v
    t[82] = -1
    t[2:53:10] = [5, 6, 7, 8, v // 3, v // 2]
    x[42] = -np.inf
    x[42, t[42]] = 2.0
    t[309], t[308] = v - 1, 0
    x = K.rounded(x, dtype)
    want, wg = K.token_loss(x, t, reduction="none")
    lb, gb = K.token_loss_bounds(x, t, -100, "none", 1.0, chain(v), dtype)
    X, T = put(rt, x, dtype), rt.Tensor.from_numpy(t)
    loss, stats = rt.softmax_cross_entropy(X, T, reduction="none")
    near(loss.to_numpy(), want, lb)
    flagged()
    up = rt.Tensor.from_numpy(np.ones(n, np.float32))
    near(get(rt.softmax_cross_entropy_backward(up, X, T, stats, reduction="none")), wg, gb)
    flagged()
    shift, _ = shifted(rt, x, dtype, 1)
    loss, _ = rt.softmax_cross_entropy(shift, T, reduction="none")
    near(loss.to_numpy(), want, lb)
    flagged()
    # the mean over those that give a number
    t[~np.isfinite(want)] = -100
    T = rt.Tensor.from_numpy(t)
    want, wg = K.token_loss(x, t)
    lb, gb = K.token_loss_bounds(x, t, -100, "mean", 1.0, chain(v), dtype)
    loss, stats = rt.softmax_cross_entropy(X, T)
    near(loss.to_numpy(), want, lb)
    near(get(rt.softmax_cross_entropy_backward(rt.Tensor.from_numpy(np.float32([1])), X, T, stats)), wg, gb)
    loss, _ = rt.softmax_cross_entropy_grad(X, T, grad=X)
    near(loss.to_numpy(), want, lb)
    near(get(X), wg, gb)
    no_flag()


@pytest.mark.parametrize("v", [3, 100, 511, 1023, 2047])
def test_loss_gradient_of_many_short_rows(rt, v):
    n = 1003
    x, t = logits_of(n, v, v, "float32")
    want, wg = K.token_loss(x, t)
    lb, gb = K.token_loss_bounds(x, t, -100, "mean", 1.0, chain(v), "float32")
    X, T = rt.Tensor.from_numpy(x), rt.Tensor.from_numpy(t)
    loss, stats = rt.softmax_cross_entropy(X, T)
    near(loss.to_numpy(), want, lb)
    near(rt.softmax_cross_entropy_backward(rt.Tensor.from_numpy(np.float32([1])), X, T, stats).to_numpy(), wg, gb)


def test_loss_without_rows(rt):
    X, T = rt.Tensor([0, 5]), rt.Tensor([0], dtype="int64")
    loss, grad = rt.softmax_cross_entropy_grad(X, T)
    assert float(loss.to_numpy().reshape(())) == 0.0 and grad.shape() == [0, 5]
    loss, _ = rt.softmax_cross_entropy(X, T, reduction="sum")
    assert float(loss.to_numpy().reshape(())) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 1000, 50257])
def test_loss_of_misaligned_tensors(rt, v, dtype):
    x, t = logits_of(4, v, 11, dtype)
    want, wg = K.token_loss(x, t)
    lb, gb = K.token_loss_bounds(x, t, -100, "mean", 1.0, chain(v), dtype)
    T = rt.Tensor.from_numpy(t)
    for a, b in ((1, 1), (3, 0), (0, 3), (1, 2)):       # logits and gradient shifted alike, and not
        X, xbuf = shifted(rt, x, dtype, a)
        G, gbuf = shifted(rt, np.zeros_like(x), dtype, b)
        loss, _ = rt.softmax_cross_entropy_grad(X, T, grad=G)
        near(loss.to_numpy(), want, lb)
        near(get(G), wg, gb)
        around = get(gbuf)
        assert (around[:b] == 9).all() and (around[b + x.size:] == 9).all()
        loss, stats = rt.softmax_cross_entropy(X, T)
        near(loss.to_numpy(), want, lb)
        rt.softmax_cross_entropy_backward(rt.Tensor.from_numpy(np.float32([1])), X, T, stats, out=G)
        near(get(G), wg, gb)


def test_loss_gradient_against_differences(rt):
    """(L(x + h) - L(x - h)) / 2h against the gradient, h = 2^-5: the loss's third
    derivative is below 1, so the difference is off by h^2/6 < 2^-12, and the
    losses (below 8, bounded by 2^-20 of error) add 2 * 2^-20 / 2h = 2^-15."""
    x, t = logits_of(2, 12, 21, "float32", masked=False)
    x = np.round(x * 64) / 64          # so that x + h and x - h are exact
    T = rt.Tensor.from_numpy(t)
    _, grad = rt.softmax_cross_entropy_grad(rt.Tensor.from_numpy(x.astype(np.float32)), T, reduction="sum")
    grad, h = grad.to_numpy(), 2.0 ** -5
    for i in range(2):
        for j in range(12):
            two = []
            for s in (h, -h):
                y = x.copy()
                y[i, j] += s
                two.append(float(rt.softmax_cross_entropy(rt.Tensor.from_numpy(y.astype(np.float32)), T, reduction="sum")[0].to_numpy().reshape(())))
            assert abs((two[0] - two[1]) / (2 * h) - grad[i, j]) <= 2.0 ** -12 + 2.0 ** -15 + 2.0 ** -20


def test_loss_is_the_same_every_time(rt):
    x, t = logits_of(500, 3001, 6, "bfloat16")
    X, T = put(rt, x, "bfloat16"), rt.Tensor.from_numpy(t)
    first = [a.to_numpy() for a in rt.softmax_cross_entropy_grad(X, T)]
    for _ in range(3):
        again = [a.to_numpy() for a in rt.softmax_cross_entropy_grad(X, T)]
        for a, b in zip(first, again):
            same(a, b)


# ---- embedding ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, d, v", [(1, 1, 1), (1, 768, 50), (3, 7, 11), (8, 64, 3), (100, 33, 1000), (17, 1024, 257), (1000, 130, 77), (5, 4100, 9)])
def test_embedding(rt, n, d, v, dtype):
    rng = np.random.default_rng(n * d)
    w = K.rounded(rng.normal(0, 1, (v, d)), dtype)
    ids = rng.integers(0, v, n)
    for scale in (1.0, float(np.sqrt(d)), -0.3):
        for index in (np.int32, np.int64):
            got = rt.embedding(put(rt, w, dtype), rt.Tensor.from_numpy(ids.astype(index)), scale=scale)
            same(get(got), K.embedding(w, ids, scale, dtype))
    W, _ = shifted(rt, w, dtype, 1)
    O, big = shifted(rt, np.zeros((n, d), np.float32), dtype, 3)
    rt.embedding(W, rt.Tensor.from_numpy(ids), out=O)
    same(get(O), w[ids])
    around = get(big)
    assert (around[:3] == 9).all() and (around[3 + n * d:] == 9).all()
    no_flag()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 15, 520, 521, 1003])
def test_embedding_of_many_ids(rt, d, dtype):
    """Several rows a thread; every start modulo 16 bytes; bad ids among them."""
    n, v = 700000 // (d + 100), 37
    rng = np.random.default_rng(d)
    w = K.rounded(rng.normal(0, 1, (v, d)), dtype)
    ids = rng.integers(0, v, n)
    want = K.embedding(w, ids, 1.5, dtype)
    O, big = shifted(rt, np.zeros((n, d), np.float32), dtype, 1)
    for a in range(16 // N.DTYPE_BYTES[O._code]):
        W, _ = shifted(rt, w, dtype, a)
        rt.embedding(W, rt.Tensor.from_numpy(ids), scale=1.5, out=O)
        same(get(O), want)
    around = get(big)
    assert (around[:1] == 9).all() and (around[1 + n * d:] == 9).all()
    no_flag()
    ids[::11], ids[1::13] = v, -7
    got = get(rt.embedding(W, rt.Tensor.from_numpy(ids), scale=1.5))
    bad = (ids < 0) | (ids >= v)
    assert np.isnan(got[bad]).all()
    same(got[~bad], want[~bad])
    flagged()


def test_embedding_shapes_and_values(rt):
    w = np.arange(12, dtype=np.float32).reshape(4, 3)
    w[1, 1], w[2, 0] = np.nan, np.inf
    W = rt.Tensor.from_numpy(w)
    ids = np.array([[3, 1], [2, 2], [0, 3]])
    out = rt.embedding(W, rt.Tensor.from_numpy(ids))
    assert out.shape() == [3, 2, 3]
    same(out.to_numpy(), w[ids])
    out = rt.embedding(W, rt.Tensor.from_numpy(np.int32(2)))
    assert out.shape() == [3]
    same(out.to_numpy(), w[2])
    assert rt.embedding(W, rt.Tensor([0], dtype="int64")).shape() == [0, 3]


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_of_bad_ids(rt, dtype):
    w = K.rounded(np.ones((10, 24)), dtype)
    ids = np.array([0, 10, 9, -1, 1 << 40, -(1 << 40), 5])
    out = get(rt.embedding(put(rt, w, dtype), rt.Tensor.from_numpy(ids)))
    good = [0, 2, 6]
    assert (out[good] == 1).all() and np.isnan(np.delete(out, good, 0)).all()
    flagged()
    g = put(rt, np.ones((7, 24)), dtype)
    gw = rt.embedding_backward(g, rt.Tensor.from_numpy(ids), 10).to_numpy()
    flagged()
    want = np.zeros((10, 24))
    want[[0, 9, 5]] = 1
    assert (gw == want).all()


GRADS = [(1, 1, 1), (1, 768, 50), (3, 7, 11), (64, 64, 3), (100, 33, 1000), (317, 1024, 257), (5000, 130, 77), (2000, 260, 70000), (9, 4100, 9),
         (40000, 8, 5), (3000, 96, 3000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, d, v", GRADS)
def test_embedding_gradient(rt, n, d, v, dtype):
    rng = np.random.default_rng(n + d + v)
    ids = np.minimum((np.exp(rng.random(n) * np.log(v + 1)) - 1).astype(np.int64), v - 1)
    g = K.rounded(rng.normal(0, 1, (n, d)), dtype)
    scale = float(np.sqrt(d))
    G, I = put(rt, g, dtype), rt.Tensor.from_numpy(ids if n % 2 else ids.astype(np.int32))
    for padding in (None, 0, v - 1):
        want, bound = K.embedding_grad(g, ids, v, scale, padding)
        near(rt.embedding_backward(G, I, v, scale=scale, padding_idx=padding).to_numpy(), want, bound + 2.0 ** -24 * np.abs(want))
        # added to what is there; rows without a token keep their bits, NaN and all
        start = rng.normal(0, 1, (v, d)).astype(np.float32)
        count = np.bincount(ids[ids != (-1 if padding is None else padding)], minlength=v)
        if (count == 0).any():
            start[np.flatnonzero(count == 0)[0]] = np.nan
        acc = rt.Tensor.from_numpy(start)
        rt.embedding_backward(G, I, v, scale=scale, padding_idx=padding, accumulate=True, out=acc)
        got = acc.to_numpy()
        same(got[count == 0], start[count == 0])
        near(got[count > 0], (start + want)[count > 0], (bound + 2.0 ** -23 * (np.abs(want) + np.abs(start)))[count > 0])
    if dtype != "float32":      # the table's gradient in the type of the activations
        want, bound = K.embedding_grad(g, ids, v, 0.5)
        out = put(rt, np.ones((v, d)), dtype)
        rt.embedding_backward(G, I, v, scale=0.5, out=out)
        half = K.half_step(dtype)
        near(get(out), want, bound * (1 + half) + np.abs(want) * (half + 2.0 ** -24) + K.least(dtype))
        rt.embedding_backward(G, I, v, scale=0.5, accumulate=True, out=out)
        first = K.rounded(want, dtype).astype(np.float64)
        near(get(out), 2 * want, 2 * bound + np.abs(want) * half * 4 + np.abs(first) * 2.0 ** -22 + 2 * K.least(dtype))
    no_flag()


@pytest.mark.parametrize("n", [255, 2048, 4095, 4096, 4097, 4609, 8193, 33000, 49151, 49152, 49153])
@pytest.mark.parametrize("kind", ["apart", "text", "padded"])
def test_embedding_gradient_of_as_many_ids(rt, n, kind):
    """Each way to sort, each length of a piece."""
    rng = np.random.default_rng(n)
    v, d = 9000, 20
    ids = np.resize(rng.permutation(v), n) if kind == "apart" else np.minimum((np.exp(rng.random(n) * np.log(v + 1)) - 1).astype(np.int64), v - 1)
    if kind == "padded":
        ids[rng.random(n) < 0.9] = 3
    g = rng.normal(0, 1, (n, d)).astype(np.float32)
    for padding in (None, 3):
        want, bound = K.embedding_grad(g, ids, v, 2.0, padding)
        G, I = rt.Tensor.from_numpy(g), rt.Tensor.from_numpy(ids)
        got = rt.embedding_backward(G, I, v, scale=2.0, padding_idx=padding)
        near(got.to_numpy(), want, bound + 2.0 ** -24 * np.abs(want))
        # added to zeros: the same sums in the same order, however the ids were sorted
        acc = rt.Tensor.from_numpy(np.zeros((v, d), np.float32))
        rt.embedding_backward(G, I, v, scale=2.0, padding_idx=padding, accumulate=True, out=acc)
        assert (acc.to_numpy() == got.to_numpy()).all()
    no_flag()


@pytest.mark.parametrize("n", [1, 31, 32, 33, 1023, 1024, 1025, 30000])
def test_embedding_gradient_of_one_id(rt, n):
    """Every token the same: one long sum."""
    rng = np.random.default_rng(n)
    g = rng.normal(0, 1, (n, 36)).astype(np.float32)
    ids = np.full(n, 7)
    want, bound = K.embedding_grad(g, ids, 20, 1.0)
    near(rt.embedding_backward(rt.Tensor.from_numpy(g), rt.Tensor.from_numpy(ids), 20).to_numpy(), want, bound)


@pytest.mark.parametrize("a, b", [(1, 1), (2, 0), (0, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_gradient_of_misaligned_tensors(rt, a, b, dtype):
    rng = np.random.default_rng(1)
    ids = rng.integers(0, 40, 90)
    g = K.rounded(rng.normal(0, 1, (90, 64)), dtype)
    G, _ = shifted(rt, g, dtype, a)
    O, big = shifted(rt, np.zeros((40, 64), np.float32), "float32", b)
    want, bound = K.embedding_grad(g, ids, 40, 1.0)
    rt.embedding_backward(G, rt.Tensor.from_numpy(ids), 40, out=O)
    near(O.to_numpy(), want, bound)
    around = big.to_numpy()
    assert (around[:b] == 9).all() and (around[b + want.size:] == 9).all()


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("v, d", [(1, 1), (6, 1), (5, 3), (13, 1), (4, 31)])
def test_embedding_gradient_of_small_tables_anywhere(rt, v, d, dtype):
    """Every start modulo 16 bytes: all of the table is written, nothing around it."""
    g = K.rounded(np.arange(1, d + 1, dtype=np.float32)[None], dtype)
    G, I = put(rt, g, dtype), rt.Tensor.from_numpy(np.array([v // 2]))
    want = np.zeros((v, d), np.float32)
    want[v // 2] = g
    for b in range(16 // N.DTYPE_BYTES[G._code]):
        O, big = shifted(rt, np.full((v, d), 5.0), dtype, b)
        rt.embedding_backward(G, I, v, out=O)
        same(get(O), want)
        around = get(big)
        assert (around[:b] == 9).all() and (around[b + want.size:] == 9).all()


def test_embedding_gradient_without_ids(rt):
    out = rt.Tensor.from_numpy(np.ones((5, 6), np.float32))
    rt.embedding_backward(rt.Tensor([0, 6]), rt.Tensor([0], dtype="int64"), 5, accumulate=True, out=out)
    assert (out.to_numpy() == 1).all()
    rt.embedding_backward(rt.Tensor([0, 6]), rt.Tensor([0], dtype="int64"), 5, out=out)
    assert (out.to_numpy() == 0).all()


def test_embedding_gradient_is_the_same_every_time(rt):
    rng = np.random.default_rng(12)
    ids = np.minimum((np.exp(rng.random(20000) * np.log(501)) - 1).astype(np.int64), 499)
    G, I = rt.Tensor.from_numpy(rng.normal(0, 1, (20000, 100)).astype(np.float32)), rt.Tensor.from_numpy(ids)
    first = rt.embedding_backward(G, I, 500).to_numpy()
    for _ in range(4):
        same(rt.embedding_backward(G, I, 500).to_numpy(), first)


# ---- AdamW over many tensors ---------------------------------------------------------

HYPER = (1e-3, 0.9, 0.999, 1e-8, 0.01)
SIZES = [[1], [127], [128], [129], [4096], [4097], [3, 5, 7], [0], [12289], [64, 64], [100003]]


def adam_state(rng, shape, gtype):
    n = int(np.prod(shape))
    return [rng.normal(0, 0.02, n).astype(np.float32).reshape(shape), K.rounded(rng.normal(0, 1e-2, n), gtype).reshape(shape),
            rng.normal(0, 1e-3, n).astype(np.float32).reshape(shape), (rng.random(n) * 1e-4).astype(np.float32).reshape(shape)]


@pytest.mark.parametrize("gtype", DTYPES)
@pytest.mark.parametrize("wd", [0.0, 0.01])
def test_adamw_multi_equals_one_by_one(rt, gtype, wd):
    rng = np.random.default_rng(4)
    host = [adam_state(rng, s, gtype) for s in SIZES]
    host[4][1][7] = np.nan
    host[4][1][8] = np.inf
    lr, b1, b2, eps, _ = HYPER
    dev = [[put(rt, a, gtype if k == 1 else "float32") for k, a in enumerate(h)] for h in host]
    copies = [rt.Tensor(s, dtype="float16" if i % 2 else "bfloat16") for i, s in enumerate(SIZES)]
    lists = [rt.TensorList([d[k] for d in dev]) for k in range(4)]
    for t in (1, 2, 1000):
        want = [rt.adamw_update(*(rt.Tensor.from_numpy(a) for a in h), lr, b1, b2, eps, wd, t) for h in host]
        rt.adamw_update_multi(*lists, lr, b1, b2, eps, wd, t, copies=copies)
        for i, (h, w) in enumerate(zip(host, want)):
            for k, a in zip((0, 2, 3), w):
                same(dev[i][k].to_numpy(), a.to_numpy())
                h[k] = a.to_numpy()
            same(get(copies[i]), K.rounded(h[0], copies[i].dtype))
            same(get(dev[i][1]), h[1])


def test_adamw_multi_of_very_many_tensors(rt):
    """More tensors than one launch takes, a plain list, misaligned ones among them."""
    rng = np.random.default_rng(9)
    host = [adam_state(rng, [int(n)], "float32") for n in rng.integers(1, 300, 1000)]
    keep, dev = [], []
    for i, h in enumerate(host):
        row = []
        for a in h:
            t, big = shifted(rt, a, "float32", i % 4)
            row.append(t)
            keep.append(big)
        dev.append(row)
    rt.adamw_update_multi(*([d[k] for d in dev] for k in range(4)), *HYPER, 3)
    flat = [np.concatenate([h[k] for h in host]) for k in range(4)]
    want = rt.adamw_update(*(rt.Tensor.from_numpy(a) for a in flat), *HYPER, 3)
    for k, w in zip((0, 2, 3), want):
        same(np.concatenate([d[k].to_numpy() for d in dev]), w.to_numpy())
    for i, big in enumerate(keep):
        a = big.to_numpy()
        o = (i // 4) % 4
        assert (a[:o] == 9).all() and (a[-8:] == 9).all()


def eight(rt, host):
    """The codes and scales of a tensor's moments, on the GPU and here."""
    m, v = host[2].ravel(), host[3].ravel()
    mc, ms = K.encode(m, None, False)
    vc, vs = K.encode(np.sqrt(v), None, True)
    shape = host[2].shape
    dev = [rt.Tensor.from_numpy(mc.reshape(shape), dtype="float8_e4m3"), rt.Tensor.from_numpy(ms),
           rt.Tensor.from_numpy(vc.reshape(shape), dtype="float8_e4m3"), rt.Tensor.from_numpy(vs)]
    return dev, [mc, ms, vc, vs]


@pytest.mark.parametrize("gtype", DTYPES)
def test_adamw_multi_in_8_bits(rt, gtype):
    """Every operation that leads to the codes is one IEEE rounding, so three
    steps' moments agree bit for bit; the parameters within the quotient's 2 ulp."""
    rng = np.random.default_rng(14)
    host = [adam_state(rng, s, gtype) for s in SIZES]
    host[4][3][100:400] *= 1e-12          # blocks of small and of widely spread moments
    host[4][2][500:600] = 0.0
    host[5][3][::3] *= 1e-9
    host[5][1][128:256] = 0.0
    host[5][2][128:256] = 0.0
    host[5][3][128:256] = 0.0
    dev8, host8 = zip(*(eight(rt, h) for h in host))
    P, G = [put(rt, h[0]) for h in host], [put(rt, h[1], gtype) for h in host]
    copies = [rt.Tensor(s, dtype="bfloat16") for s in SIZES]
    host8 = list(host8)
    for t in (1, 2, 700):
        rt.adamw_update_multi(P, G, [d[0] for d in dev8], [d[2] for d in dev8], *HYPER, t, m_scales=[d[1] for d in dev8],
                              v_scales=[d[3] for d in dev8], copies=copies, seed=t * 10 ** 12)
        for i, h in enumerate(host):
            p, bound, *codes = K.adamw8(h[0].ravel(), h[1].ravel(), *host8[i], *HYPER, t, t * 10 ** 12, i)
            host8[i] = codes
            h[0] = P[i].to_numpy()
            near(h[0].ravel(), p, bound)
            same(get(copies[i]), K.bf16(h[0]))
            for d, w in zip(dev8[i], codes):
                assert (d.to_numpy().ravel() == w).all()


def test_adamw_multi_in_8_bits_of_values_that_are_not_finite(rt):
    rng = np.random.default_rng(15)
    h = adam_state(rng, [256], "float32")
    h[1][3], h[1][70], h[1][200] = np.nan, np.inf, 1e30      # v = 1e57 overflows, m does not
    dev, codes = eight(rt, h)
    P, G = put(rt, h[0]), put(rt, h[1])
    rt.adamw_update_multi([P], [G], [dev[0]], [dev[2]], *HYPER, 1, m_scales=[dev[1]], v_scales=[dev[3]], seed=5)
    p, bound, *want = K.adamw8(h[0], h[1], *codes, *HYPER, 1, 5, 0)
    near(P.to_numpy(), p, np.nan_to_num(bound))
    for d, w in zip(dev, want):
        assert (d.to_numpy() == w).all()
    v = K.decode(dev[2].to_numpy(), dev[3].to_numpy())
    assert np.isnan(v[[3, 70, 200]]).all() and np.isfinite(np.delete(v, [3, 70, 200])).all()
    assert (np.delete(v, [3, 70, 200]) > 0).all()            # never 0: nothing divides by eps alone


def test_adamw_multi_in_8_bits_misaligned_and_reseeded(rt):
    rng = np.random.default_rng(16)
    n = 1000
    h = adam_state(rng, [n], "bfloat16")
    outs = []
    for seed, off in ((1, 0), (1, 1), (2, 0), (1, 3)):
        dev, codes = eight(rt, h)
        P, pb = shifted(rt, h[0], "float32", off)
        G, gb = shifted(rt, h[1], "bfloat16", off)
        raw = rt.Tensor.from_numpy(np.concatenate([np.zeros(off, np.uint8), codes[0]]), dtype="float8_e4m3")
        M = rt.Tensor.from_device_ptr(raw.ptr + off, [n], owner=raw, dtype="float8_e4m3")
        rt.adamw_update_multi([P], [G], [M], [dev[2]], *HYPER, 4, m_scales=[dev[1]], v_scales=[dev[3]], seed=seed)
        outs.append((P.to_numpy(), M.to_numpy(), dev[2].to_numpy()))
    for k in range(3):
        assert (outs[0][k] == outs[1][k]).all() and (outs[0][k] == outs[3][k]).all()
    assert (outs[0][1] != outs[2][1]).any()                   # another seed, another rounding


def test_adamw8_pack_and_unpack(rt):
    rng = np.random.default_rng(17)
    for n in (1, 127, 128, 129, 5000):
        m, v = rng.normal(0, 1e-3, n).astype(np.float32), (rng.random(n) * 1e-4).astype(np.float32) ** 3
        m[0], v[0] = 0.0, 0.0
        mc, ms, vc, vs = rt.adamw8_pack(rt.Tensor.from_numpy(m), rt.Tensor.from_numpy(v))
        wmc, wms = K.encode(m, None, False)
        wvc, wvs = K.encode(np.sqrt(v), None, True)
        for a, b in ((mc, wmc), (ms, wms), (vc, wvc), (vs, wvs)):
            assert (a.to_numpy() == b).all()
        bm, bv = rt.adamw8_unpack(mc, ms, vc, vs)
        same(bm.to_numpy(), K.decode(wmc, wms))
        same(bv.to_numpy(), K.decode(wvc, wvs) ** 2)


# ---- together, and other streams ------------------------------------------------------

def bigram(rt, steps, bits, table, ids, targets):
    """A bigram model: the logits of a token's successor are its row of the
    table.  One training step is the embedding, the loss with its gradient, the
    table's gradient and AdamW."""
    v = table.shape[0]
    W, B = rt.Tensor.from_numpy(table), rt.Tensor.from_numpy(np.zeros(v, np.float32))
    I, T = rt.Tensor.from_numpy(ids), rt.Tensor.from_numpy(targets)
    moments = [[rt.Tensor.zeros(t.shape()), rt.Tensor.zeros(t.shape())] for t in (W, B)]
    scales = None
    if bits == 8:
        packed = [rt.adamw8_pack(*p) for p in moments]
        moments, scales = [[p[0], p[2]] for p in packed], [[p[1], p[3]] for p in packed]
    losses = []
    for t in range(1, steps + 1):
        logits = rt.add_broadcast(rt.embedding(W, I), B)
        loss, dx = rt.softmax_cross_entropy_grad(logits, T, grad=logits)
        dw = rt.embedding_backward(dx, I, v)
        db = rt.sum_dim(dx, 0)
        rt.adamw_update_multi([W, B], [dw, db], [p[0] for p in moments], [p[1] for p in moments], 0.05, 0.9, 0.99, 1e-8, 0.01, t,
                              m_scales=scales and [p[0] for p in scales], v_scales=scales and [p[1] for p in scales], seed=t)
        losses.append(float(loss.to_numpy().reshape(())))
    return losses, W.to_numpy(), B.to_numpy()


def bigram_plain(steps, table, ids, targets):
    w, b = table.astype(np.float64), np.zeros(table.shape[0])
    m, s = [np.zeros_like(w), np.zeros_like(b)], [np.zeros_like(w), np.zeros_like(b)]
    losses = []
    for t in range(1, steps + 1):
        loss, dx = K.token_loss(w[ids] + b, targets)
        dw = np.zeros_like(w)
        np.add.at(dw, ids, dx)
        for k, (p, g) in enumerate(((w, dw), (b, dx.sum(0)))):
            m[k] = 0.9 * m[k] + 0.1 * g
            s[k] = 0.99 * s[k] + 0.01 * g * g
            old = p.copy()
            p -= 0.05 * (m[k] / (1 - 0.9 ** t)) / (np.sqrt(s[k] / (1 - 0.99 ** t)) + 1e-8) + 0.05 * 0.01 * old
        losses.append(loss)
    return losses, w, b


def bigram_data():
    rng = np.random.default_rng(30)
    v, n = 61, 400
    ids = rng.integers(0, v, n)
    targets = (ids * 7 + rng.integers(0, 3, n)) % v
    targets[::11] = -100
    return rng.normal(0, 0.1, (v, v)).astype(np.float32), ids, targets


def test_a_bigram_model_trains(rt):
    """Eight steps against 64 bits.  Adam's quotient m/sqrt(v) is near 1 whatever
    the gradient's size, so a gradient's relative error d moves a step by at most
    lr * 2d; gradients here are sums of at most 400 terms (2^-24 * 400 of them,
    2^-15; those of the least rows cancel little as only the target's is
    negative), which over 8 steps of 0.05 is 2^-15 * 2 * 8 * 0.05 < 2^-14."""
    table, ids, targets = bigram_data()
    losses, w, b = bigram(rt, 8, 32, table, ids, targets)
    want, ww, wb = bigram_plain(8, table, ids, targets)
    assert np.abs(np.array(losses) - want).max() <= 2.0 ** -13
    assert np.abs(w - ww).max() <= 2.0 ** -14 and np.abs(b - wb).max() <= 2.0 ** -14


def test_a_bigram_model_trains_in_8_bits(rt):
    table, ids, targets = bigram_data()
    losses, w, b = bigram(rt, 8, 8, table, ids, targets)
    again = bigram(rt, 8, 8, table, ids, targets)
    assert np.isfinite(losses).all() and np.isfinite(w).all()
    assert losses == again[0] and (w == again[1]).all()       # the seeds decide the rounding


def run_all(rt, s):
    """Every token operator once, on the calling thread's stream."""
    rt.embedding(s["w"], s["ids"], scale=2.0, out=s["emb"])
    rt.softmax_cross_entropy(s["x"], s["t"], loss=s["loss1"], stats=s["stats"])
    rt.softmax_cross_entropy_backward(s["up"], s["x"], s["t"], s["stats"], out=s["g1"])
    rt.softmax_cross_entropy_grad(s["x"], s["t"], loss=s["loss2"], grad=s["g2"])
    rt.embedding_backward(s["emb"], s["ids"], s["w"].shape()[0], out=s["dw"])
    rt.embedding_backward(s["emb"], s["ids"], s["w"].shape()[0], accumulate=True, out=s["dw"])
    rt.adamw_update_multi([s["p"]], [s["dw"]], [s["m"]], [s["v"]], *HYPER, 2)
    rt.adamw_update_multi([s["p8"]], [s["dw"]], [s["m8"]], [s["v8"]], *HYPER, 2, m_scales=[s["ms"]], v_scales=[s["vs"]], seed=1)


def state_for_all(rt, seed):
    rng = np.random.default_rng(seed)
    f = lambda *shape: rt.Tensor.from_numpy(rng.normal(0, 1, shape).astype(np.float32))  # noqa: E731
    v, d, n, c = 700, 96, 3000, 1234
    s = {"w": f(v, d), "ids": rt.Tensor.from_numpy(rng.integers(0, v, n)), "emb": f(n, d), "x": f(n, c),
         "t": rt.Tensor.from_numpy(rng.integers(0, c, n)), "loss1": f(1), "loss2": f(1), "stats": f(n, 3), "g1": f(n, c),
         "g2": f(n, c), "up": f(1), "dw": f(v, d), "p": f(v, d), "m": f(v, d), "v": rt.Tensor.from_numpy(rng.random((v, d)).astype(np.float32)),
         "p8": f(v, d)}
    s["m8"], s["ms"], s["v8"], s["vs"] = rt.adamw8_pack(s["m"], s["v"])
    return s


RESULTS = ("emb", "loss1", "loss2", "g1", "g2", "dw", "p", "m", "v", "p8", "m8", "ms", "v8", "vs")


def results(s):
    return [s[k].to_numpy() for k in RESULTS]


@pytest.mark.parametrize("kind", ["stream", "thread"])
def test_on_another_stream(rt, kind):
    import threading
    torch = pytest.importorskip("torch")
    a, b = state_for_all(rt, 3), state_for_all(rt, 3)
    run_all(rt, a)
    want = results(a)
    N.check(N.lib().rtc_synchronize())
    stream = torch.cuda.Stream()

    def work():
        N.check(N.lib().rtc_set_stream(ctypes.c_void_p(stream.cuda_stream) if kind == "stream" else None))
        try:
            run_all(rt, b)
            N.check(N.lib().rtc_synchronize())
        finally:
            N.check(N.lib().rtc_set_stream(None))

    if kind == "stream":
        work()
    else:
        t = threading.Thread(target=work)
        t.start()
        t.join()
    for x, y in zip(results(b), want):
        assert (x == y).all()


def test_captured_into_graphs(rt):
    """Two graphs over different state, replayed in turn and at once; each call's
    scratch is its own."""
    torch = pytest.importorskip("torch")
    states = [state_for_all(rt, 5), state_for_all(rt, 6)]
    plain = [state_for_all(rt, 5), state_for_all(rt, 6)]
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, stream in zip(states, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            N.check(N.lib().rtc_set_stream(ctypes.c_void_p(stream.cuda_stream)))
            try:
                run_all(rt, s)
            finally:
                N.check(N.lib().rtc_set_stream(None))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for s in plain:
            run_all(rt, s)
        N.check(N.lib().rtc_synchronize())
        for s, w in zip(states, plain):
            for x, y in zip(results(s), results(w)):
                assert (x == y).all()
    del graphs


def test_two_calls_at_once(rt):
    """Two streams, no waiting between them."""
    torch = pytest.importorskip("torch")
    states, plain = [state_for_all(rt, 7), state_for_all(rt, 8)], [state_for_all(rt, 7), state_for_all(rt, 8)]
    for s in plain:
        run_all(rt, s)
    N.check(N.lib().rtc_synchronize())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        for s, stream in zip(states, streams):
            N.check(N.lib().rtc_set_stream(ctypes.c_void_p(stream.cuda_stream)))
            run_all(rt, s)
    finally:
        N.check(N.lib().rtc_set_stream(None))
    torch.cuda.synchronize()
    for s, w in zip(states, plain):
        for x, y in zip(results(s), results(w)):
            assert (x == y).all()


FIRST = """
import ctypes, sys
import torch
import rusttorch_b200 as rt
from rusttorch_b200 import _native as N
f = lambda *shape, t=torch.float32: (torch.rand(shape, device="cuda") * 40).to(t)
def wrap(x):
    name = {torch.float32: "float32", torch.int64: "int64", torch.uint8: "float8_e4m3"}[x.dtype]
    return rt.Tensor.from_device_ptr(x.data_ptr(), x.shape, owner=x, dtype=name)
w, emb, loss, p, gr, m, v = f(50, 8), f(300, 8), f(1), f(400), f(400), f(400), f(400)
x, g = f(300, 9000), f(300, 9000)
ids, mc, vc, ms, vs = f(300, t=torch.int64), f(400, t=torch.uint8), f(400, t=torch.uint8), f(4), f(4)
W, E, I, X, L, G, P, GR, M, V, MC, VC, MS, VS = map(wrap, (w, emb, ids, x, loss, g, p, gr, m, v, mc, vc, ms, vs))
h = (1e-3, 0.9, 0.999, 1e-8, 0.01, 1)
call = {
    "embedding": lambda: rt.embedding(W, I, out=E),
    "embedding_backward": lambda: rt.embedding_backward(E, I, 50, out=W),
    "softmax_cross_entropy_grad": lambda: rt.softmax_cross_entropy_grad(X, I, loss=L, grad=G),
    "adamw_update_multi": lambda: rt.adamw_update_multi([P], [GR], [M], [V], *h),
    "adamw_update_multi_8": lambda: rt.adamw_update_multi([P], [GR], [MC], [VC], *h, m_scales=[MS], v_scales=[VS], seed=3),
}[sys.argv[1]]
outputs = (w, emb, loss, p, m, v, g, mc, vc, ms, vs)
start = [y.clone() for y in outputs]
stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=stream):
    N.check(N.lib().rtc_set_stream(ctypes.c_void_p(stream.cuda_stream)))
    call()
    N.check(N.lib().rtc_set_stream(None))
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outputs, start)), "it ran while it was captured"
graph.replay()
torch.cuda.synchronize()
got = [y.clone() for y in outputs]
assert not all(torch.equal(a, b) for a, b in zip(got, start))
for y, a in zip(outputs, start):
    y.copy_(a)
torch.cuda.synchronize()
call()
N.check(N.lib().rtc_synchronize())
assert all(torch.equal(a, b) for a, b in zip(outputs, got))
del graph
print("fine")
"""


@pytest.mark.parametrize("op", ["embedding", "embedding_backward", "softmax_cross_entropy_grad",
                                "adamw_update_multi", "adamw_update_multi_8"])
def test_first_call_of_a_process_is_captured(op):
    """Nothing that a first call sets up may need a stream that is not capturing."""
    import subprocess
    import sys
    from pathlib import Path
    pytest.importorskip("torch")
    r = subprocess.run([sys.executable, "-c", FIRST, op], cwd=Path(__file__).resolve().parents[1],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stderr[-2000:]


def test_two_threads_at_once(rt):
    import threading
    torch = pytest.importorskip("torch")
    states, plain = [state_for_all(rt, 9), state_for_all(rt, 10)], [state_for_all(rt, 9), state_for_all(rt, 10)]
    for s in plain:
        for _ in range(20):
            run_all(rt, s)
    N.check(N.lib().rtc_synchronize())
    errors = []

    def work(s, stream):
        try:
            N.check(N.lib().rtc_set_stream(ctypes.c_void_p(stream.cuda_stream)))
            for _ in range(20):
                run_all(rt, s)
            N.check(N.lib().rtc_synchronize())
        except Exception as e:
            errors.append(e)
        finally:
            N.check(N.lib().rtc_set_stream(None))

    threads = [threading.Thread(target=work, args=(s, torch.cuda.Stream())) for s in states]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s, w in zip(states, plain):
        for x, y in zip(results(s), results(w)):
            assert (x == y).all()


def wrap(rt, x, dtype):
    return rt.Tensor.from_device_ptr(x.data_ptr(), x.shape, owner=x, dtype=dtype)


def test_embedding_past_32_bits(rt):
    """More than 2^32 elements: the last rows, and sums that are whole numbers."""
    torch = pytest.importorskip("torch")
    n, d, v = (1 << 20) + 12345, 4096, 300
    ids = torch.arange(n, device="cuda") * 7 % v
    w = torch.arange(v, device="cuda").repeat_interleave(d).reshape(v, d).to(torch.bfloat16)
    out = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    rt.embedding(wrap(rt, w, "bfloat16"), wrap(rt, ids, "int64"), out=wrap(rt, out, "bfloat16"))
    no_flag()
    for rows in (slice(0, 5), slice((1 << 20) - 3, (1 << 20) + 3), slice(n - 5, n)):
        assert torch.equal(out[rows], w[ids[rows]])
    out.fill_(1.0)
    torch.cuda.synchronize()
    gw = rt.embedding_backward(wrap(rt, out, "bfloat16"), wrap(rt, ids, "int64"), v).to_numpy()
    no_flag()
    count = np.bincount(ids.cpu().numpy(), minlength=v)
    assert (gw == count[:, None]).all()


def test_loss_past_32_bits(rt):
    """Equal logits, more than 2^32 of them: loss log V, gradient 1/V and 1/V - 1."""
    torch = pytest.importorskip("torch")
    n, v = 33000, 131072
    x = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    t = torch.arange(n, device="cuda") % v
    loss, stats = torch.empty(n, device="cuda"), torch.empty(n, 3, device="cuda")
    torch.cuda.synchronize()
    X, T, L, S = wrap(rt, x, "bfloat16"), wrap(rt, t, "int64"), wrap(rt, loss, "float32"), wrap(rt, stats, "float32")
    rt.softmax_cross_entropy(X, T, reduction="none", loss=L, stats=S)
    rt.synchronize()
    # 17 log 2: the log's error and the rounding, 2^-22 each of it
    assert float((loss.double() - 17 * np.log(2)).abs().max()) <= 17 * np.log(2) * 2.0 ** -21
    loss.zero_()
    torch.cuda.synchronize()
    rt.softmax_cross_entropy_grad(X, T, reduction="none", loss=L, grad=X)
    no_flag()
    assert float((loss.double() - 17 * np.log(2)).abs().max()) <= 17 * np.log(2) * 2.0 ** -21
    for i in (0, 1, 32767, 32768, n - 1):
        row = x[i].double()
        assert float(row[i]) == -1.0                 # 2^-17 - 1 in bfloat16
        row[i] = 2.0 ** -17
        assert bool((row == 2.0 ** -17).all())


# ---- reports of bad ids -------------------------------------------------------------------

def reported():
    """Whether rtc_synchronize reports a bad id."""
    try:
        N.check(N.lib().rtc_synchronize())
        return 0
    except N.RusttorchError as e:
        assert e.code == N.INVALID_ARGUMENT and "outside the vocabulary" in str(e)
        return 1


def test_a_bad_id_is_reported_beside_a_wait_that_ran_out(rt):
    W, I, O = rt.Tensor.from_numpy(np.ones((4, 8), np.float32)), rt.Tensor.from_numpy(np.array([9])), rt.Tensor([1, 8])
    no_flag()
    N.check(N.lib().rtc_selftest_bounded_wait())
    rt.embedding(W, I, out=O)
    with pytest.raises(N.RusttorchError) as e:
        N.check(N.lib().rtc_synchronize())
    assert e.value.code == N.BACKEND_ERROR and "gave up waiting" in str(e.value)
    flagged()


def test_every_bad_id_is_reported_once_while_another_thread_asks(rt):
    """One thread meets a bad id in each of its rounds and asks at the round's
    end; another, on a stream of its own, asks all the time.  Whoever asks
    first gets the report: one for each round, none lost and none twice."""
    import threading
    torch = pytest.importorskip("torch")
    W, I, O = rt.Tensor.from_numpy(np.ones((4, 8), np.float32)), rt.Tensor.from_numpy(np.array([9])), rt.Tensor([1, 8])
    no_flag()
    rounds, done, errors, reports = 1000, threading.Event(), [], [0, 0]

    def work(k, stream):
        try:
            N.check(N.lib().rtc_set_stream(ctypes.c_void_p(stream.cuda_stream)))
            if k == 0:
                for _ in range(rounds):
                    rt.embedding(W, I, out=O)
                    reports[0] += reported()
            else:
                while not done.is_set():
                    reports[1] += reported()
        except BaseException as e:
            errors.append(e)
        finally:
            N.check(N.lib().rtc_set_stream(None))
            if k == 0:
                done.set()

    threads = [threading.Thread(target=work, args=(k, torch.cuda.Stream())) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert sum(reports) + reported() == rounds, reports


# ---- how close the loss's terms are -----------------------------------------------------------

@pytest.mark.parametrize("n, v", [(3, 1000), (5, 1003), (700, 260), (3, 50257), (400, 9000), (2, 300001), (2, 600001)])
def test_f32_loss_gradient_is_as_close_as_softmax(rt, n, v):
    """Within softmax's 1e-6 for unlikely tokens too: the maximum is 20.5 and every
    other logit 30 to 86 below it on a grid of 2^-10, so that x_j - M is exact.
    A gradient is off by its term's 2^y (2^-22) and that one's last sum (2^-24),
    the product with 1/s and upstream (2^-24 each of the two), 1/s (2^-24), and s,
    whose largest term, 1, is within 3.1 * 2^-23 and whose others are less than
    v e^-30 < 2^-24 together, lost or not: 16 * 2^-24 = 9.6e-7 covers these.  In
    the target's, -o/s, what o and s have in common cancels."""
    rng = np.random.default_rng(v)
    d = np.round(rng.uniform(30, 86, (n, v)) * 1024) / 1024
    c, t = rng.integers(0, v, n), rng.integers(0, v, n)
    t = np.where(t == c, (t + 1) % v, t)
    d[np.arange(n), c] = 0
    x = (20.5 - d).astype(np.float32)
    assert (20.5 - x.astype(np.float64) == d).all()
    want, wg = K.token_loss(x, t, reduction="none")
    one, T = rt.Tensor.from_numpy(np.ones(n, np.float32)), rt.Tensor.from_numpy(t)
    for X in (rt.Tensor.from_numpy(x), shifted(rt, x, "float32", 1)[0]):
        loss, grad = rt.softmax_cross_entropy_grad(X, T, reduction="none")
        near(grad.to_numpy(), wg, 16 * 2.0 ** -24 * np.abs(wg))
        loss, stats = rt.softmax_cross_entropy(X, T, reduction="none")
        near(rt.softmax_cross_entropy_backward(one, X, T, stats, reduction="none").to_numpy(), wg, 16 * 2.0 ** -24 * np.abs(wg))
    no_flag()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_16_bit_loss_terms(rt, dtype):
    """Two classes a row that are not ruled out, the target the larger: the loss is
    log1p(e^-d).  The term is within (0.62 d + 3.1) 2^-23 of itself, which log1p
    passes on at most, and log1p within 2 ulp, 2^-22."""
    rng = np.random.default_rng(8)
    n, v = 4000, 16
    top = K.rounded(rng.uniform(-400, 400, n), dtype)
    low = K.rounded(top - np.where(np.arange(n) % 2, rng.uniform(0, 2, n), rng.uniform(0, 80, n)).astype(np.float32), dtype)
    top, low = np.maximum(top, low).astype(np.float64), np.minimum(top, low).astype(np.float64)
    a = rng.integers(0, v, n)
    b = (a + rng.integers(1, v, n)) % v
    x = np.full((n, v), -np.inf, np.float32)
    x[np.arange(n), a], x[np.arange(n), b] = top, low
    d = top - low
    want = np.log1p(np.exp(-d))
    loss, _ = rt.softmax_cross_entropy(put(rt, x, dtype), rt.Tensor.from_numpy(a), reduction="none")
    near(loss.to_numpy(), want, want * ((0.62 * d + 3.1) * 2.0 ** -23 + 2.0 ** -22))
    loss, _ = rt.softmax_cross_entropy_grad(put(rt, x, dtype), rt.Tensor.from_numpy(a), reduction="none")
    near(loss.to_numpy(), want, want * ((0.62 * d + 3.1) * 2.0 ** -23 + 2.0 ** -22))


# ---- more than one turn: buffers in turn, passes of the sort, tables of tensors ---------------

def eight_bit_step(rt, host, gtypes, ctypes_, offsets, hyper, t, seed):
    """One 8-bit step of `host`'s tensors, every code, scale and copy bit for bit and
    the parameters within their bound; tensor i starts offsets[i] elements into its buffer."""
    P, G, M, V, MS, VS, C, codes, keep = [], [], [], [], [], [], [], [], []
    for h, gtype, ctype, off in zip(host, gtypes, ctypes_, offsets):
        dev, here = eight(rt, h)
        for k, (a, kind) in enumerate(((h[0], "float32"), (h[1], gtype))):
            x, big = shifted(rt, a, kind, off)
            (P, G)[k].append(x)
            keep.append(big)
        M.append(dev[0]), MS.append(dev[1]), V.append(dev[2]), VS.append(dev[3])
        C.append(rt.Tensor(h[0].shape, dtype=ctype))
        codes.append(here)
    rt.adamw_update_multi(P, G, M, V, *hyper, t, m_scales=MS, v_scales=VS, copies=C, seed=seed)
    for i, h in enumerate(host):
        want, bound, *after = K.adamw8(h[0].ravel(), h[1].ravel(), *codes[i], *hyper, t, seed, i)
        got = P[i].to_numpy()
        near(got.ravel(), want, bound)
        same(get(C[i]), K.rounded(got, C[i].dtype))
        for d, w in zip((M[i], MS[i], V[i], VS[i]), after):
            assert (d.to_numpy().ravel() == w).all(), i
    for big, off in zip(keep, np.repeat(offsets, 2)):
        a = get(big)
        assert (a[:off] == 9).all() and (a[-8:] == 9).all()


@pytest.mark.parametrize("wd", [0.0, 0.01])
def test_adamw_multi_in_8_bits_of_many_units(rt, wd):
    """5.9 million elements are 2880 units of 2048: six and more to each of the
    3 * 148 blocks at most that are resident, so that every buffer of a block's three
    is filled twice and each barrier passes both its phases; whole units and parts of
    one, tensors that are not aligned, empty ones between, each type of gradient and copy."""
    rng = np.random.default_rng(40)
    sizes = [2_200_000, 0, 1_300_001, 2047, 700_003, 128, 900_000, 800_129, 1]
    host = [adam_state(rng, [n], DTYPES[i % 3]) for i, n in enumerate(sizes)]
    host[0][2][500_000:500_100] = 0.0
    host[2][3][::3] *= 1e-9                 # values under the format's normal range
    eight_bit_step(rt, host, [DTYPES[i % 3] for i in range(9)], [DTYPES[1 + i // 2 % 2] for i in range(9)],
                   [0, 0, 0, 0, 1, 0, 0, 3, 0], (1e-3, 0.9, 0.999, 1e-8, wd), 7, 3 << 40)


@pytest.mark.parametrize("n", [100, 900])
def test_adamw_multi_in_8_bits_of_very_many_tensors(rt, n):
    """Lists for the larger arguments of the kernel, and for three launches."""
    rng = np.random.default_rng(n)
    host = [adam_state(rng, [int(s)], "bfloat16") for s in rng.integers(0, 400, n)]
    eight_bit_step(rt, host, ["bfloat16"] * n, ["float16"] * n, [(0, 0, 0, 5)[i % 4] for i in range(n)], HYPER, 3, 77)


def test_adamw_multi_in_8_bits_past_32_bits(rt):
    """A tensor of more than 2^32 elements: its last ones, whose random bits count on."""
    torch = pytest.importorskip("torch")
    n, last = (1 << 32) + 70001, 70001 + 300          # whole blocks of 128, and a part, on both sides of 2^32
    begin = (n - last) // K.BLOCK * K.BLOCK
    last = n - begin
    rng = np.random.default_rng(41)
    tail = rng.normal(0, 1e-2, last).astype(np.float32)
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 2.0 ** -7, dtype=torch.bfloat16, device="cuda")
    tail = K.bf16(tail)
    g[begin:] = torch.from_numpy(tail).cuda().to(torch.bfloat16)
    codes, scales = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)], [torch.zeros(-(-n // K.BLOCK), device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    W = lambda x, kind: [wrap(rt, x, kind)]
    rt.adamw_update_multi(W(p, "float32"), W(g, "bfloat16"), W(codes[0], "float8_e4m3"), W(codes[1], "float8_e4m3"), *HYPER, 1,
                          m_scales=W(scales[0], "float32"), v_scales=W(scales[1], "float32"), seed=9)
    no_flag()
    i = np.arange(begin, n, dtype=np.uint64)
    with np.errstate(over="ignore"):
        bits = K.mix32(np.uint32(K.tensor_key(9, 0)) + i.astype(np.uint32) * np.uint32(0x9E3779B1) + (i >> np.uint64(32)).astype(np.uint32) * np.uint32(0xBB67AE85))
    one = np.float32(1)
    m = tail * (one - np.float32(0.9))
    r = np.sqrt((tail * tail) * (one - np.float32(0.999)))
    for x, least, low, k in ((m, False, bits & np.uint32(0xffff), 0), (r, True, bits >> np.uint32(16), 1)):
        c, s = K.encode(x, low, least)
        assert (codes[k][begin:].cpu().numpy() == c).all()
        assert (scales[k][begin // K.BLOCK:].cpu().numpy() == s).all()
    # the first ones: all gradients alike, so the first step moves each by lr, to the digits of two quotients
    assert float((p[:1 << 20] + 1e-3).abs().max()) <= 1e-3 * (2.0 ** -20 + 1e-8 / (2.0 ** -7 * 0.03))
    del p, g, codes, scales
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n", [5000, 40000, 60001])
@pytest.mark.parametrize("v, d", [(50257, 3), (131072, 2), (300000, 2), ((1 << 27) + 9, 1)])
def test_embedding_gradient_of_large_vocabularies(rt, n, v, d):
    """Two passes of 8 and 9 bits, three and four: whole numbers, so that sums are exact."""
    rng = np.random.default_rng(n + d)
    ids = rng.integers(0, v, n)
    ids[::5] = ids[3]                                 # one that is frequent
    ids[1::50] = v - 1 - rng.integers(0, 3, len(ids[1::50]))
    ids[2], ids[n - 1] = 0, v - 1
    g = rng.integers(-8, 9, (n, d)).astype(np.float32)
    named, at = np.unique(ids, return_inverse=True)
    want = np.zeros((len(named), d))
    np.add.at(want, at, g)
    G, I = rt.Tensor.from_numpy(g), rt.Tensor.from_numpy(ids)
    for padding in (None, v - 1):
        w = np.where((named == padding)[:, None], 0, want) if padding is not None else want
        out = rt.embedding_backward(G, I, v, padding_idx=padding)
        got = out.to_numpy()
        assert (got[named] == w).all()
        got[named] = 0
        assert not got.any()
        # added to it: twice as much
        rt.embedding_backward(G, I, v, padding_idx=padding, accumulate=True, out=out)
        got = out.to_numpy()
        assert (got[named] == 2 * w).all()
        got[named] = 0
        assert not got.any()
    no_flag()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n, v", [(7200, 1000), (3600, 2500), (1800, 5000), (100, 120001)])
def test_loss_and_gradient_of_several_rows_a_block(rt, n, v, dtype):
    """Three rows and more to each block (or cluster) that can be resident, for each
    size of block, ignored rows among them: both buffers, each barrier's phases."""
    v *= 1 if dtype == "float32" else 2               # the same bytes to a row
    x, t = logits_of(n, v, n, dtype)
    rng = np.random.default_rng(n)
    t[rng.random(n) < 0.3] = -100
    t[n // 2:n // 2 + n // 10] = -100
    want, wg = K.token_loss(x, t, reduction="none")
    lb, gb = K.token_loss_bounds(x, t, -100, "none", 1.0, chain(v), dtype)
    X, T = put(rt, x, dtype), rt.Tensor.from_numpy(t)
    loss, grad = rt.softmax_cross_entropy_grad(X, T, reduction="none")
    near(loss.to_numpy(), want, lb)
    near(get(grad), wg, gb)
    loss, grad = rt.softmax_cross_entropy_grad(X, T, reduction="none", grad=X)
    near(loss.to_numpy(), want, lb)
    near(get(X), wg, gb)
    no_flag()


def test_a_bigram_model_moves_alike_in_8_bits(rt):
    """The first step starts from moments of 0, which 8 bits hold exactly: both forms
    move a parameter alike but for the roundings of their quotients, 16 of 2^-24 in
    all (8 operations in f32's, and 8 in the other's with 2^-23 for the reciprocal's),
    and half an ulp of the parameter in each of the two differences on both sides."""
    table, ids, targets = bigram_data()
    losses, w, b = bigram(rt, 1, 32, table, ids, targets)
    losses8, w8, b8 = bigram(rt, 1, 8, table, ids, targets)
    assert losses == losses8
    for start, x, y in ((table, w, w8), (np.zeros_like(b), b, b8)):
        move = np.abs(x.astype(np.float64) - start)
        assert (move > 0.04).any()
        near(y, x, 0.05 * 2.0 ** -20 + np.abs(start) * 2.0 ** -22 + np.abs(x) * 2.0 ** -22)


# ---- after an error --------------------------------------------------------------------------

def test_a_call_after_one_that_ran_out_of_memory(rt):
    """An error is reported by the call that met it, and by no later one."""
    x = rt.Tensor.from_numpy(np.arange(8, dtype=np.float32))
    W, I, O = rt.Tensor.from_numpy(np.ones((4, 8), np.float32)), rt.Tensor.from_numpy(np.array([9, 1])), rt.Tensor([2, 8])
    no_flag()

    def fails():
        with pytest.raises(N.RusttorchError) as e:
            rt.Tensor([1 << 45])
        assert e.value.code == N.BACKEND_ERROR and "MemoryAllocation" in str(e.value)

    fails()
    same(rt.add(x, x).to_numpy(), np.arange(0, 16, 2))
    fails()
    rt.embedding(W, I, out=O)
    fails()
    flagged()
    same(O.to_numpy()[1], np.ones(8))
    G = rt.Tensor.from_numpy(np.ones((2, 8), np.float32))
    fails()
    out = rt.Tensor([4, 8])
    fails()
    rt.embedding_backward(G, rt.Tensor.from_numpy(np.array([2, 2])), 4, out=out)
    same(out.to_numpy(), np.repeat([[0], [0], [2], [0]], 8, 1))
    no_flag()
