"""The token operators and AdamW over many tensors on the CPU: refusals (all
before any CUDA call; descriptors point at dummy addresses) and the arithmetic
of the 8-bit moments."""
import ctypes

import numpy as np
import pytest

from rusttorch_b200 import _native as N
from tests import _tokens as K

A, B, C, D, E, F = (0x10000000 * k for k in range(1, 7))


def desc(shape, dtype=N.F32, device=0, ptr=A):
    return N.Desc(ptr, shape, dtype, device)


def call(name, *args):
    args = [a.ref if isinstance(a, N.Desc) else a for a in args]
    res = getattr(N.lib(), name)(*args)
    if res.success:
        return None
    msg = ctypes.string_at(res.error_msg).decode()
    N.lib().rtc_free_error_message(res.error_msg)
    return res.code, msg


def array(*descs):
    arr = (N.RtcTensor * len(descs))()
    for i, d in enumerate(descs):
        arr[i] = d.s
    arr._keep = descs
    return arr


# ---- embedding -------------------------------------------------------------------

W, IDS, OUT = dict(shape=[10, 4], ptr=A), dict(shape=[3], dtype=N.I64, ptr=B), dict(shape=[3, 4], ptr=C)


@pytest.mark.parametrize("change, code, text", [
    (dict(w=dict(dtype=N.F64)), N.DTYPE_MISMATCH, "embedding (weight): expected float32, bfloat16 or float16, got float64"),
    (dict(ids=dict(dtype=N.F32)), N.DTYPE_MISMATCH, "embedding (ids): expected int32 or int64, got float32"),
    (dict(out=dict(dtype=N.BF16)), N.DTYPE_MISMATCH, "embedding (output): expected float32, got bfloat16"),
    (dict(w=dict(shape=[40])), N.INVALID_ARGUMENT, "two dimensions"),
    (dict(out=dict(shape=[3, 5])), N.SHAPE_MISMATCH, "expected [3, 4], got [3, 5]"),
    (dict(out=dict(shape=[4])), N.SHAPE_MISMATCH, "expected [3, 4], got [4]"),
    (dict(out=dict(device=1)), N.INVALID_ARGUMENT, "same device"),
    (dict(ids=dict(device=-1)), N.INVALID_ARGUMENT, "ids must be a device tensor"),
    (dict(ids=dict(device=-2)), N.INVALID_ARGUMENT, "invalid device"),
    (dict(out=dict(ptr=A + 16)), N.INVALID_ARGUMENT, "must not overlap"),
    (dict(out=dict(ptr=B)), N.INVALID_ARGUMENT, "must not overlap"),
    (dict(out=dict(ptr=C + 2)), N.INVALID_ARGUMENT, "aligned to its element type"),
    (dict(ids=dict(ptr=0)), N.INVALID_ARGUMENT, "data must not be null"),
    (dict(w=dict(dtype=7)), N.INVALID_ARGUMENT, "Unknown dtype code: 7"),
])
def test_embedding_refusals(change, code, text):
    w, ids, out = (desc(**{**base, **change.get(k, {})}) for k, base in (("w", W), ("ids", IDS), ("out", OUT)))
    got = call("rtc_embedding", w, ids, 1.0, out)
    assert got is not None and got[0] == code and text in got[1], got


def test_embedding_of_nothing_needs_no_gpu():
    assert call("rtc_embedding", desc([10, 4]), desc([0], N.I64, ptr=0), 1.0, desc([0, 4], ptr=0)) is None
    assert call("rtc_embedding", desc([10, 0], ptr=0), desc([3], N.I32, ptr=B), 1.0, desc([3, 0], ptr=0)) is None


def test_strided_tensors_are_refused():
    w = desc([10, 4])
    w.s.strides = (ctypes.c_size_t * 2)(8, 1)
    got = call("rtc_embedding", w, desc(**IDS), 1.0, desc(**OUT))
    assert got[0] == N.UNSUPPORTED and "non-contiguous" in got[1]


@pytest.mark.parametrize("change, padding, code, text", [
    (dict(gw=dict(dtype=N.F16)), -1, N.DTYPE_MISMATCH, "expected float32 or bfloat16, got float16"),
    (dict(g=dict(dtype=N.I64)), -1, N.DTYPE_MISMATCH, "(grad_output)"),
    (dict(ids=dict(dtype=N.BF16)), -1, N.DTYPE_MISMATCH, "(ids)"),
    (dict(gw=dict(shape=[10, 5])), -1, N.SHAPE_MISMATCH, "expected [3, 5], got [3, 4]"),
    (dict(gw=dict(shape=[10, 4, 1])), -1, N.INVALID_ARGUMENT, "two dimensions"),
    (dict(), 10, N.INVALID_ARGUMENT, "below the number of rows (10), got 10"),
    (dict(gw=dict(ptr=B)), -1, N.INVALID_ARGUMENT, "must not overlap"),
    (dict(gw=dict(ptr=C + 8)), -1, N.INVALID_ARGUMENT, "must not overlap"),
    (dict(g=dict(shape=[1 << 31, 4]), ids=dict(shape=[1 << 31])), -1, N.INVALID_ARGUMENT, "fewer than 2^31"),
])
def test_embedding_backward_refusals(change, padding, code, text):
    g, ids, gw = (desc(**{**base, **change.get(k, {})}) for k, base in
                  (("g", dict(shape=[3, 4], dtype=N.BF16, ptr=C)), ("ids", IDS), ("gw", dict(shape=[10, 4], ptr=D * 100))))
    got = call("rtc_embedding_backward", g, ids, 1.0, padding, 0, gw)
    assert got is not None and got[0] == code and text in got[1], got


# ---- loss ------------------------------------------------------------------------

X, T, L, S, G = (dict(shape=[3, 8], dtype=N.BF16, ptr=A), dict(shape=[3], dtype=N.I32, ptr=B), dict(shape=[], ptr=C),
                 dict(shape=[3, 3], ptr=D), dict(shape=[3, 8], dtype=N.BF16, ptr=E))


@pytest.mark.parametrize("change, reduction, code, text", [
    (dict(x=dict(dtype=N.I32)), 1, N.DTYPE_MISMATCH, "(logits)"),
    (dict(t=dict(dtype=N.F32)), 1, N.DTYPE_MISMATCH, "(targets): expected int32 or int64, got float32"),
    (dict(t=dict(shape=[4])), 1, N.SHAPE_MISMATCH, "expected [4, 8], got [3, 8]"),
    (dict(x=dict(shape=[]), t=dict(shape=[])), 1, N.INVALID_ARGUMENT, "last dimension"),
    (dict(x=dict(shape=[3, 0], ptr=0), g=dict(shape=[3, 0], ptr=0)), 1, N.EMPTY_TENSOR, "empty tensor"),
    (dict(l=dict(shape=[3])), 1, N.INVALID_ARGUMENT, "must have one element, got 3"),
    (dict(), 0, N.SHAPE_MISMATCH, "expected [3], got []"),
    (dict(), 3, N.INVALID_ARGUMENT, "'reduction'"),
    (dict(l=dict(dtype=N.BF16)), 1, N.DTYPE_MISMATCH, "expected float32, got bfloat16"),
    (dict(l=dict(ptr=A)), 1, N.INVALID_ARGUMENT, "must not overlap"),
    (dict(s=dict(shape=[3, 2])), 1, N.SHAPE_MISMATCH, "expected [3, 3], got [3, 2]"),
    (dict(s=dict(ptr=A + 4)), 1, N.INVALID_ARGUMENT, "must not overlap"),
    (dict(s=dict(device=1)), 1, N.INVALID_ARGUMENT, "same device"),
])
def test_softmax_cross_entropy_refusals(change, reduction, code, text):
    x, t, l, s = (desc(**{**base, **change.get(k, {})}) for k, base in (("x", X), ("t", T), ("l", L), ("s", S)))
    got = call("rtc_softmax_cross_entropy", x, t, -100, reduction, l, s)
    assert got is not None and got[0] == code and text in got[1], got
    if not ("s" in change):
        g = desc(**{**G, **change.get("g", {})})
        fused = call("rtc_softmax_cross_entropy_grad", x, t, -100, reduction, 1.0, l, g)
        assert fused is not None and fused[0] == code, fused


@pytest.mark.parametrize("change, code, text", [
    (dict(g=dict(dtype=N.F32)), N.DTYPE_MISMATCH, "expected bfloat16, got float32"),
    (dict(g=dict(shape=[3, 9])), N.SHAPE_MISMATCH, "(grad_logits)"),
    (dict(g=dict(ptr=A + 16)), N.INVALID_ARGUMENT, "must not overlap"),
    (dict(g=dict(ptr=B)), N.INVALID_ARGUMENT, "must not overlap"),
    (dict(g=dict(ptr=C)), N.INVALID_ARGUMENT, "must not overlap"),
    (dict(g=dict(ptr=D)), N.INVALID_ARGUMENT, "must not overlap"),
    (dict(s=dict(shape=[9])), N.SHAPE_MISMATCH, "(stats)"),
    (dict(l=dict(shape=[2])), N.INVALID_ARGUMENT, "one element"),
])
def test_softmax_cross_entropy_backward_refusals(change, code, text):
    x, t, l, s, g = (desc(**{**base, **change.get(k, {})}) for k, base in
                     (("x", X), ("t", T), ("l", L), ("s", S), ("g", G)))
    got = call("rtc_softmax_cross_entropy_backward", l, x, t, s, -100, 1, g)
    assert got is not None and got[0] == code and text in got[1], got


def test_loss_without_rows():
    x, t, l = desc([0, 8], ptr=0), desc([0], N.I64, ptr=0), desc([0], ptr=0)
    assert call("rtc_softmax_cross_entropy", x, t, -100, 0, l, None) is None


def test_other_ops_refuse_the_new_types():
    for code in (N.BF16, N.F16, N.F8E4M3):
        got = call("rtc_relu", desc([4], code), desc([4], code))
        assert got == (N.INVALID_ARGUMENT, f"Invalid argument 'dtype': Unknown dtype code: {code}")


# ---- AdamW over many tensors -------------------------------------------------------

def multi(p, g, m, v, ms=None, vs=None, copies=None, n=None, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, t=1):
    lists = [array(*x) if x is not None else None for x in (p, g, m, v, ms, vs, copies)]
    return call("rtc_adamw_update_multi", *lists, len(p) if n is None else n, lr, b1, b2, eps, wd, t, 0)


def four(n=256, base=A, dtype=N.F32, moments=N.F32):
    return [[desc([n], d, ptr=base + 0x100000 * k)] for k, d in enumerate((N.F32, dtype, moments, moments))]


def test_no_tensors_is_no_work():
    assert call("rtc_adamw_update_multi", None, None, None, None, None, None, None, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 0) is None


@pytest.mark.parametrize("kw, text", [
    (dict(lr=-1.0), "'learning_rate': must be positive, got -1"),
    (dict(b1=1.0), "'beta1': must be in (0, 1), got 1"),
    (dict(b2=0.0), "'beta2': must be in (0, 1), got 0"),
    (dict(eps=0.0), "'epsilon': must be positive, got 0"),
    (dict(wd=-0.5), "'weight_decay': must be non-negative, got -0.5"),
    (dict(t=0), "'timestep': must be >= 1"),
])
def test_adamw_multi_hyperparameters(kw, text):
    code, msg = multi(*four(), **kw)
    assert code == N.INVALID_ARGUMENT and text in msg


def test_adamw_multi_names_the_tensor_at_fault():
    p, g, m, v = four()
    q, h, k, w = four(base=B)
    h = [desc([255], ptr=B + 0x100000)]
    code, msg = multi(p + q, g + h, m + k, v + w)
    assert code == N.SHAPE_MISMATCH and "grads[1]" in msg and "expected [256], got [255]" in msg
    q = [desc([256], N.BF16, ptr=B)]
    code, msg = multi(p + q, g + g, m + m, v + v)
    assert code == N.DTYPE_MISMATCH and "params[1]" in msg
    code, msg = multi(p, g, m, v, copies=[desc([256], N.F32, ptr=C)])
    assert code == N.DTYPE_MISMATCH and "copies[0]: expected bfloat16 or float16" in msg


def test_adamw_multi_refuses_shared_memory():
    p, g, m, v = four()
    q, h, k, w = four(base=B)
    for lists in ((p + p, g + h, m + k, v + w),            # a parameter twice
                  (p, p, m, v),                            # the gradient is the parameter
                  (p + q, g + h, m + m, v + w),            # shared moments
                  (p, g, m, m)):
        code, msg = multi(*lists)
        assert code == N.INVALID_ARGUMENT and "must not overlap another tensor of the call" in msg
    inside = [desc([256], ptr=A + 64)]
    code, msg = multi(p + inside, g + h, m + k, v + w)
    assert code == N.INVALID_ARGUMENT and "must not overlap" in msg
    code, msg = multi(p, g, m, v, copies=[desc([256], N.BF16, ptr=A + 1020)])
    assert code == N.INVALID_ARGUMENT and "must not overlap" in msg


def test_adamw_multi_moment_types():
    p, g, m, v = four(moments=N.F8E4M3)
    code, msg = multi(p, g, m, v)
    assert code == N.DTYPE_MISMATCH and "m[0]: expected float32" in msg
    ms, vs = [desc([2], ptr=C)], [desc([2], ptr=D)]
    code, msg = multi(p, g, m, v, ms=ms)
    assert code == N.INVALID_ARGUMENT and "both" in msg
    code, msg = multi(p, g, m, v, ms=[desc([3], ptr=C)], vs=vs)
    assert code == N.INVALID_ARGUMENT and "m_scales[0]" in msg and "(2), got 3" in msg
    p, g, m, v = four()
    code, msg = multi(p, g, m, v, ms=ms, vs=vs)
    assert code == N.DTYPE_MISMATCH and "m[0]: expected float8_e4m3, got float32" in msg


def test_adamw_multi_too_many_tensors():
    code, msg = multi(*four(), n=(1 << 20) + 1)
    assert code == N.INVALID_ARGUMENT and "at most" in msg


def test_adamw8_pack_refusals():
    m, v, mc, vc = desc([200], ptr=A), desc([200], ptr=B), desc([200], N.F8E4M3, ptr=C), desc([200], N.F8E4M3, ptr=D)
    ms, vs = desc([2], ptr=E), desc([2], ptr=F)
    assert call("rtc_adamw8_pack", m, desc([201], ptr=B), mc, ms, vc, vs)[0] == N.SHAPE_MISMATCH
    assert call("rtc_adamw8_pack", m, v, m, ms, vc, vs)[0] == N.DTYPE_MISMATCH
    assert call("rtc_adamw8_pack", m, v, mc, desc([1], ptr=E), vc, vs)[0] == N.INVALID_ARGUMENT
    assert call("rtc_adamw8_pack", m, v, mc, ms, desc([200], N.F8E4M3, ptr=C), vs)[0] == N.INVALID_ARGUMENT
    assert call("rtc_adamw8_unpack", mc, ms, vc, ms, m, v)[0] == N.INVALID_ARGUMENT


def test_python_refusals():
    import rusttorch_b200 as rt
    t = rt.Tensor([4], ptr=0x1000)
    with pytest.raises(ValueError):
        rt.Tensor([4], ptr=0x1000, dtype="float8")
    with pytest.raises(ValueError):
        rt.softmax_cross_entropy(t, t, reduction="max")
    with pytest.raises(ValueError):
        rt.adamw_update_multi([t, t], [t], [t, t], [t, t], 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    with pytest.raises(ValueError):
        rt.embedding_backward(t, t, 4, accumulate=True)
    with pytest.raises(rt.RusttorchError):
        rt.embedding_backward(t, t, 4, out=rt.Tensor([3, 4], ptr=0x1000))
    with pytest.raises(rt.RusttorchError):
        rt.Tensor.from_numpy(np.zeros(3))
    with pytest.raises(rt.RusttorchError):
        rt.Tensor.from_numpy(np.zeros(3, np.float32), dtype="float16")


def test_no_float64_tensors():
    """No operator takes them, so none is made: not by name, not from an array."""
    import rusttorch_b200 as rt
    with pytest.raises(ValueError, match="dtype must be one of .*not 'float64'"):
        rt.Tensor([4], ptr=0x1000, dtype="float64")
    with pytest.raises(ValueError, match="not 'float64'"):
        rt.Tensor.from_device_ptr(0x1000, [4], dtype="float64")
    with pytest.raises(rt.RusttorchError):
        rt.Tensor.from_numpy(np.zeros(3), dtype="float64")


# ---- the 8-bit moments' arithmetic --------------------------------------------------

def test_e4m3_table():
    assert K.E4M3[0x7e] == 448 and K.E4M3[1] == 2.0 ** -9 and K.E4M3[8] == 2.0 ** -6 and np.isnan(K.E4M3[0xff])
    assert (np.diff(K.E4M3[:0x7f]) > 0).all()
    codes = np.arange(0x7f, dtype=np.uint8)
    assert (K.to_code(K.E4M3[codes]) == codes).all()


def test_stochastic_rounding_is_unbiased():
    """Over all 2^16 random values the mean of the rounded value is the value:
    off by at most 2^-16 of a step (the bits' resolution, centred), plus, below
    2^-6, the f32 rounding of y + 2^-6 (2^-30 of it, 2^-21 of a step)."""
    bits = np.arange(1 << 16, dtype=np.uint32)
    rng = np.random.default_rng(3)
    for y in np.concatenate([2.0 ** rng.uniform(-12, 8.8, 40), K.E4M3[1:0x7f:9]]).astype(np.float32):
        z = K.round_up_or_down(np.full(1 << 16, y, np.float32), bits).astype(np.float64)
        step = 2.0 ** (max(np.floor(np.log2(float(y))), -6) - 3)
        assert set(np.unique(z)) <= set(K.E4M3[:0x7f].astype(np.float64))
        assert abs(z.mean() - float(y)) <= step * (2.0 ** -16 + 2.0 ** -21)


def test_random_bits_are_spread():
    """Means of n uniform values of 16 bits stay within 5 standard deviations,
    sqrt(1/12n), of 1/2 (2^16 values of (i + 1/2)/2^16 have that mean), for
    both halves; and the two halves are uncorrelated to 5/sqrt(n)."""
    n = 1 << 20
    for key in (0, 1, 0x12345678, K.tensor_key(7, 3)):
        with np.errstate(over="ignore"):
            h = K.mix32(np.uint32(key) + np.arange(n, dtype=np.uint32) * np.uint32(0x9E3779B1))
        lo, hi = ((h & 0xffff) + 0.5) / 65536, ((h >> 16) + 0.5) / 65536
        for u in (lo, hi):
            assert abs(u.mean() - 0.5) < 5 * np.sqrt(1 / (12 * n))
            assert abs(np.corrcoef(u[1:], u[:-1])[0, 1]) < 5 / np.sqrt(n)
        assert abs(np.corrcoef(lo, hi)[0, 1]) < 5 / np.sqrt(n)


def test_average_follows_its_input_in_8_bits():
    """v = 0.999^6 v + (1 - 0.999^6) g^2 moves by 0.6 % a step, far less than a
    code's width (6 to 12 % of sqrt(v), 12 to 26 % of v), so that rounding to
    nearest would leave it where it starts, 100 times g^2.  After 1000 steps
    exact arithmetic has g^2 (1 + 99 * 0.999^6000).  The rounding keeps sqrt(v)'s
    mean; what is left is the curvature of sqrt(b r^2 + c) over the codes that r is
    spread over: spread by at most a step or so (1/8 of r), half of its square,
    1 %, and the mean of 4096 elements is off by (1/8)/64 = 0.2 %.  5 % is thrice
    their sum; a stuck average is off by a factor of 9."""
    n, b2 = 4096, 0.999 ** 6
    mc, ms = K.encode(np.zeros(n, np.float32), None, False)
    vc, vs = K.encode(np.full(n, 1.0, np.float32), None, True)
    p, g = np.zeros(n, np.float32), np.full(n, 0.1, np.float32)
    for t in range(1, 1001):
        p, _, mc, ms, vc, vs = K.adamw8(p, g, mc, ms, vc, vs, 1e-3, 0.9, b2, 1e-8, 0.0, t, t, 0)
    root = K.decode(vc, vs).astype(np.float64)
    assert abs(root.mean() / np.sqrt(0.01 * (1 + 99 * b2 ** 1000)) - 1) < 0.05


def test_rounding_to_nearest_would_not_follow():
    """The reason for the stochastic rounding: the codes of 0.999 v to nearest
    are v's own (each moves sqrt(v) by 0.05 %, half a step is 3 %)."""
    r = K.E4M3[8:0x7f]
    assert (K.to_code(r * np.float32(np.sqrt(0.999))) == np.arange(8, 0x7f)).all()
