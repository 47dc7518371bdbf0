"""Plain 64-bit (and, for the 8-bit moments, step-by-step f32) forms of the
token operators and AdamW over many tensors, for their tests."""
import numpy as np

F32 = np.float32


def bf16(a):
    """float32 values rounded to bfloat16, as float32."""
    a = np.ascontiguousarray(a, F32)
    b = a.view(np.uint32)
    r = ((b + np.uint32(0x7fff) + ((b >> 16) & 1)) & np.uint32(0xffff0000)).view(F32)
    return np.where(np.isnan(a), F32(np.nan), r)


def rounded(a, dtype):
    """float32 values rounded to a storage type, as float32."""
    if dtype == "bfloat16":
        return bf16(a)
    with np.errstate(over="ignore"):
        return np.asarray(a, F32).astype(np.float16).astype(F32) if dtype == "float16" else np.asarray(a, F32)


def half_step(dtype):
    """The largest relative error of one rounding to a storage type."""
    return {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]


def least(dtype):
    """Half the spacing of a storage type's subnormals."""
    return {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}[dtype]


# ---- softmax cross entropy -----------------------------------------------------

def token_loss(x, targets, ignore=-100, reduction="mean", scale=1.0):
    """(loss, gradient) in 64 bits; x [N, V]."""
    x = np.asarray(x, np.float64)
    n, v = x.shape
    rows = np.zeros(n)
    grad = np.zeros((n, v))
    counted = targets != ignore
    with np.errstate(all="ignore"):
        for i in np.flatnonzero(counted):
            t = targets[i]
            if not 0 <= t < v or np.isnan(x[i]).any() or np.isposinf(x[i]).any() or np.isneginf(x[i]).all():
                rows[i] = np.nan
                grad[i] = np.nan
                continue
            top = x[i].max()
            e = np.exp(x[i] - top)
            et, e[t] = e[t], 0.0
            others = e.sum()
            s = others + et
            rows[i] = np.log1p(others) if x[i, t] == top else np.log(s) - (x[i, t] - top)
            grad[i] = e / s
            grad[i, t] = -others / s
    k = scale / max(1, counted.sum()) if reduction == "mean" else scale
    loss = rows if reduction == "none" else rows.sum() / (max(1, counted.sum()) if reduction == "mean" else 1)
    return loss, np.where(counted[:, None], grad * k, 0.0)


def token_loss_bounds(x, targets, ignore, reduction, scale, chain, dtype):
    """Largest errors of the f32 computation, (loss, gradient).

    The f32 terms e^d, d = x_j - M <= 0: d is rounded once (|d| 2^-24 of e^d),
    scaled by log2 e (as much again) and exponentiated (2 ulp, 2^-22): relative
    (|d| + 2) 2^-22 covers them.  A sum of positive terms adds `chain` roundings
    of 2^-24, the longest path of additions of any kernel.  The loss is the
    log of the sum: an absolute error of the sum's relative one, plus the
    rounding of M - x_t, of the log and of the end result (2^-22 of each).  The
    gradient adds the quotient, the factor and the product (2^-21), and the
    rounding to its type."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        d = np.where(np.isfinite(top - x), top - x, 0.0)
        e = np.exp(x - top)
        e[np.arange(len(x)), np.where((targets >= 0) & (targets < x.shape[1]), targets, 0)] *= 0
        weight = e.sum(1, keepdims=True)
        rel_sum = np.where(weight > 0, ((d + 2) * e).sum(1, keepdims=True) / weight, 2.0) * 2.0 ** -22
        rel_sum = np.nan_to_num(rel_sum) + chain * 2.0 ** -24
        loss, grad = token_loss(x, targets, ignore, "none", 1.0)
        xt = d[np.arange(len(x)), np.where((targets >= 0) & (targets < x.shape[1]), targets, 0)]
        # where the target is the maximum the loss is log1p(o) <= o: its error is relative
        row = np.where(xt == 0, np.nan_to_num(loss) * (rel_sum[:, 0] + 2.0 ** -21),
                       rel_sum[:, 0] + (np.abs(np.nan_to_num(loss)) + xt + 4) * 2.0 ** -22)
        row = np.where(targets == ignore, 0.0, row)
        count = max(1, (targets != ignore).sum())
        if reduction == "none":
            lb = row
        else:
            total = row.sum() + np.abs(np.nan_to_num(loss)).sum() * 2.0 ** -23
            lb = total / (count if reduction == "mean" else 1)
        g = np.nan_to_num(token_loss(x, targets, ignore, reduction, scale)[1])
        gb = np.abs(g) * ((d + 2) * 2.0 ** -22 + rel_sum + 2.0 ** -21 + half_step(dtype)) + least(dtype) + 2.0 ** -140
    return lb, gb


# ---- embedding -----------------------------------------------------------------

def embedding(w, ids, scale, dtype):
    """Exactly what the f32 product and one rounding give."""
    return rounded(np.asarray(w, F32)[ids] * F32(scale), dtype)


def embedding_grad(g, ids, vocab, scale, padding=None):
    """(gradient in 64 bits, bound of the f32 sum's error before the last rounding)."""
    g = np.asarray(g, np.float64).reshape(-1, g.shape[-1])
    ids = np.asarray(ids).reshape(-1)
    keep = (ids >= 0) & (ids < vocab) & (ids != (-1 if padding is None else padding))
    total = np.zeros((vocab, g.shape[1]))
    size = np.zeros((vocab, g.shape[1]))
    np.add.at(total, ids[keep], g[keep])
    np.add.at(size, ids[keep], np.abs(g[keep]))
    count = np.bincount(ids[keep], minlength=vocab)[:vocab, None]
    s = float(F32(scale))
    # count - 1 additions and the product, each off by 2^-24 of at most the sizes' sum
    return total * s, size * abs(s) * (count + 1) * 2.0 ** -24


# ---- AdamW ---------------------------------------------------------------------

E4M3 = np.array([((-1.0) ** (c >> 7)) * ((c & 7) * 2.0 ** -9 if (c >> 3) & 15 == 0 else
                                         (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7))
                 if c & 0x7f != 0x7f else np.nan for c in range(256)], F32)
BLOCK = 128


def mix32(x):
    with np.errstate(over="ignore"):
        x = np.asarray(x, np.uint32)
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
        return x ^ (x >> np.uint32(16))


def tensor_key(seed, i):
    m = (1 << 64) - 1
    z = (seed + (i + 1) * 0x9E3779B97F4A7C15) & m
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & m
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & m
    return (z ^ (z >> 31)) & 0xFFFFFFFF


def blocks(x):
    n = len(x)
    return np.pad(np.asarray(x, F32), (0, -n % BLOCK)).reshape(-1, BLOCK)


def block_scale(top):
    """Least 2^e with top <= 448 * 2^e, e >= -126, by doubling and halving in 64 bits."""
    out = []
    for t in np.asarray(top, np.float64):
        e = -126
        while t > 448 * 2.0 ** e:
            e += 1
        out.append(2.0 ** e)
    return np.array(out, F32)


def round_up_or_down(y, bits16):
    """|y| <= 448 rounded to e4m3's values, up where the part cut off plus the
    random bits (of 2^16, centred) reach a whole step."""
    low = y < 2.0 ** -6
    z = np.where(low, y + F32(2.0 ** -6), y).astype(F32)
    u = z.view(np.uint32) + (bits16.astype(np.uint32) << np.uint32(4)) + np.uint32(8)
    z = (u & np.uint32(0xfff00000)).view(F32)
    return np.where(low, z - F32(2.0 ** -6), z).astype(F32)


def to_code(z):
    """Nearest e4m3 code of z >= 0, ties to even (exact where z is a value)."""
    vals = E4M3[:0x7f].astype(np.float64)
    z = np.asarray(z, np.float64)
    hi = np.clip(np.searchsorted(vals, z), 1, 0x7e)
    lo = hi - 1
    dl, dh = z - vals[lo], vals[hi] - z
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return np.where(z <= 0, 0, c).astype(np.uint8)


def encode(x, bits16, least_code):
    """(codes, scales) of x (flat f32); bits16 None: to nearest."""
    b = blocks(x)
    size = np.abs(b)
    with np.errstate(invalid="ignore", over="ignore"):
        scale = block_scale(np.where(np.isfinite(size), size, 0).max(1))
        y = (size * (F32(1) / scale)[:, None]).astype(F32)
        fine = np.isfinite(size)
        y = np.where(fine, y, 0).astype(F32)
        z = y if bits16 is None else round_up_or_down(y, blocks_u(bits16))
    c = to_code(z)
    if least_code:
        c = np.where((c == 0) & (size > 0) & fine, 1, c)
    c = np.where(fine, c, 0x7f) | (np.signbit(b).astype(np.uint8) << 7)
    return c.reshape(-1)[:len(x)].astype(np.uint8), scale


def blocks_u(x):
    n = len(x)
    return np.pad(np.asarray(x, np.uint32), (0, -n % BLOCK)).reshape(-1, BLOCK)


def decode(codes, scales):
    return (E4M3[codes] * np.repeat(scales, BLOCK)[:len(codes)]).astype(F32)


def adamw8(p, g, mc, ms, vc, vs, lr, b1, b2, eps, wd, t, seed, index):
    """One step with 8-bit moments, every operation rounded to f32 as documented:
    (parameters, largest error of theirs, codes and scales).  The quotient is
    within 2 ulp (2^-22 of it) of the rounded one here, which its product with
    the step size passes on with a rounding of its own (2^-23 covers both
    sides'), and each of the two differences rounds at most half an ulp apart
    from a value that close: 2^-23 of the parameter each."""
    p, g = np.asarray(p, F32), np.asarray(g, F32)
    with np.errstate(all="ignore"):
        m, root = decode(mc, ms), decode(vc, vs)
        fb1, fb2 = F32(b1), F32(b2)
        m = m * fb1 + g * (F32(1) - fb1)
        v = (root * root) * fb2 + (g * g) * (F32(1) - fb2)
        r = np.sqrt(v)
        den = r * F32(1 / np.sqrt(1 - b2 ** t)) + F32(eps)
        move = (m / den) * F32(lr / (1 - b1 ** t))
        out = p - move
        if wd > 0:
            out = out - p * F32(lr * wd)
    i = np.arange(len(p), dtype=np.uint64)
    with np.errstate(over="ignore"):
        bits = mix32(np.uint32(tensor_key(seed, index)) + i.astype(np.uint32) * np.uint32(0x9E3779B1))
    mc, ms = encode(m, bits & np.uint32(0xffff), False)
    vc, vs = encode(r, bits >> np.uint32(16), True)
    assert out.dtype == F32
    with np.errstate(invalid="ignore"):
        bound = np.abs(move.astype(np.float64)) * (2.0 ** -22 + 2.0 ** -23) + (np.abs(p) + np.abs(out)).astype(np.float64) * 2.0 ** -23
    return out, bound, mc, ms, vc, vs
