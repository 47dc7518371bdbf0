"""What is measured of the token operators: the cases, their plain forms and the framework's calls.

Three families, the parts of a language model's training step that are not matrix products:

* the loss of token ids against logits, with its gradient (`softmax_cross_entropy*`);
* the embedding of token ids, with its gradient (`embedding`, `embedding_backward`);
* the AdamW step over many tensors at once, its moments in 32 bits or in 8 (`adamw_update_multi`).

Where `own` is false, `run` computes them with elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100
BLOCK = 128                      # elements that share a scale in the 8-bit moments
LR, B1, B2, EPS, WD, STEP = 1e-3, 0.9, 0.999, 1e-8, 0.01, 10


def listed():
    return [
        # one short sequence on a small vocabulary: the call's latency
        {"name": "loss_grad_small", "op": "loss_grad", "rows": 32, "vocab": 1000, "dtype": "f32"},
        # a training batch on an odd vocabulary: no row but the first starts on a 16-byte boundary
        {"name": "loss_grad_odd_bf16", "op": "loss_grad", "rows": 8192, "vocab": 50257, "dtype": "bf16"},
        # the same step in 32 bits
        {"name": "loss_grad_f32", "op": "loss_grad", "rows": 4096, "vocab": 32768, "dtype": "f32"},
        # a long batch on a large vocabulary
        {"name": "loss_grad_large_bf16", "op": "loss_grad", "rows": 8192, "vocab": 131072, "dtype": "bf16"},
        # forward, then backward from an upstream gradient, as a tape runs them; few long rows
        {"name": "loss_tape_few_rows", "op": "loss_tape", "rows": 8, "vocab": 131072, "dtype": "f32"},
        # the embedding of one decoding step
        {"name": "embed_small", "op": "embed", "rows": 8, "width": 768, "vocab": 50257, "dtype": "f32"},
        # the embedding of a training batch
        {"name": "embed_large_bf16", "op": "embed", "rows": 32768, "width": 4096, "vocab": 131072, "dtype": "bf16"},
        # the whole gradient of a table, most of whose rows no token names
        {"name": "embed_grad_dense", "op": "embed_grad", "rows": 16384, "width": 1024, "vocab": 50257, "dtype": "f32", "accumulate": False},
        # a micro-batch's gradient added to the sum of those before
        {"name": "embed_grad_accum_bf16", "op": "embed_grad", "rows": 32768, "width": 4096, "vocab": 131072, "dtype": "bf16", "accumulate": True},
        # a toy model's parameters: the call's latency
        {"name": "adamw_small", "op": "adamw", "bits": 32, "width": 64, "ff": 256, "depth": 2, "vocab": 1000, "dtype": "f32", "copy": False},
        # 194 tensors, 139 M parameters, moments in 32 bits
        {"name": "adamw_f32", "op": "adamw", "bits": 32, "width": 640, "ff": 2560, "depth": 24, "vocab": 32768, "dtype": "f32", "copy": False},
        # 98 tensors, 417 M parameters, bf16 gradients and a bf16 copy, moments in 8 bits
        {"name": "adamw_8bit_large", "op": "adamw", "bits": 8, "width": 1536, "ff": 6144, "depth": 12, "vocab": 50257, "dtype": "bf16", "copy": True},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["loss_grad", "loss_grad", "loss_tape", "embed", "embed_grad", "embed_grad", "adamw", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    size = 4 if dtype == "f32" else 2
    if op in ("loss_grad", "loss_tape"):
        vocab = log(100, 200000)
        return {"op": op, "rows": log(1, max(1, min(16384, (1 << 31) // (size * vocab)))), "vocab": vocab, "dtype": dtype}
    vocab = log(100, 131072)
    if op == "embed":
        return {"op": op, "rows": log(1, 32768), "width": log(16, 4096), "vocab": vocab, "dtype": dtype}
    if op == "embed_grad":
        return {"op": op, "rows": log(1, 32768), "width": log(16, 4096), "vocab": vocab, "dtype": dtype, "accumulate": rng.random() < 0.5}
    width = log(32, 1024)
    return {"op": op, "bits": rng.choice([8, 32]), "width": width, "ff": rng.randint(2 * width, 4 * width),
            "depth": rng.randint(1, 12), "vocab": log(100, 50257), "dtype": dtype, "copy": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _token_ids(n, vocab, gen):
    """Ids as text has them: log-uniform ranks (near Zipf's law) over a shuffled vocabulary."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)
    return torch.randperm(vocab, generator=gen, device="cuda")[rank]


def _distinct(n, vocab):
    """How many different ids _token_ids gives on average."""
    p = np.log1p(1.0 / (np.arange(vocab) + 1.0)) / math.log(vocab + 1)
    return float(np.sum(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def _sizes(case):
    """The tensors of a decoder with an untied table: per layer four square matrices, two of the feed-forward, two norms."""
    d, f = case["width"], case["ff"]
    return [case["vocab"] * d] + [d * d] * (4 * case["depth"]) + [d * f] * (2 * case["depth"]) + [d] * (2 * case["depth"] + 1)


def _layout(sizes):
    """Where each tensor starts in the flat buffer (whole blocks of BLOCK), and the buffer's length."""
    blocks = -(-np.asarray(sizes, np.int64) // BLOCK)
    ends = np.cumsum(blocks)
    return (ends - blocks) * BLOCK, blocks, int(ends[-1]) * BLOCK


def _blocks(sizes):
    """Of each block of the flat buffer: its tensor, and where in that tensor it starts."""
    _, blocks, total = _layout(sizes)
    per = torch.from_numpy(blocks).cuda()
    tensor = torch.arange(len(sizes), device="cuda").repeat_interleave(per)
    first = (per.cumsum(0) - per).repeat_interleave(per)
    return tensor, (torch.arange(total // BLOCK, device="cuda") - first) * BLOCK


def _flat(sizes, make):
    """A flat buffer of make(n)'s values with zeros between the tensors."""
    tensor, inside = _blocks(sizes)
    left = torch.tensor(sizes, device="cuda")[tensor] - inside
    return (make(len(inside) * BLOCK).view(-1, BLOCK) * (torch.arange(BLOCK, device="cuda") < left[:, None])).view(-1)


def _to_codes(x, least):
    """Moments in 8 bits to start from: e4m3 codes to nearest under a power of two for each block."""
    y = x.view(-1, BLOCK)
    scale = _scale(y.abs().amax(1))
    c = (y / scale[:, None]).to(torch.float8_e4m3fn)
    if least:
        c = torch.where(y > 0, c.float().clamp(min=2.0 ** -9), c.float()).to(torch.float8_e4m3fn)
    return c.view(-1), scale


def prepare(case, seed):
    gen = _gen(seed)
    s = dict(case)
    if case["op"] in ("loss_grad", "loss_tape"):
        n, v, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        logits = torch.empty(n, v, dtype=dt, device="cuda")
        targets = _token_ids(n, v, gen)
        for a in range(0, n, 1024):          # in parts: the values are drawn in 32 bits
            part = torch.randn(min(1024, n - a), v, generator=gen, device="cuda") * 3
            sure = torch.rand(part.shape[0], generator=gen, device="cuda") < 0.3      # tokens that the model is sure of
            part.scatter_add_(1, targets[a:a + 1024, None], torch.where(sure, 12.0, 4.0)[:, None])
            logits[a:a + 1024] = part
        logits[:, torch.randint(0, v, (max(1, v // 100),), generator=gen, device="cuda")] = -math.inf   # tokens that are ruled out
        logits.scatter_(1, targets[:, None], logits.gather(1, targets[:, None]).clamp(min=-4.0))
        if n > 1:
            targets[torch.rand(n, generator=gen, device="cuda") < 0.05] = IGNORE
            targets[0] = 0
            logits[0, 0] = 1.0
        s.update(logits=logits, targets=targets)
        if case["op"] == "loss_tape":
            s["upstream"] = torch.full((1,), 0.7, device="cuda")
    elif case["op"] == "embed":
        s["weight"] = (torch.randn(case["vocab"], case["width"], generator=gen, device="cuda") * 0.02).to(DTYPES[case["dtype"]])
        s["ids"] = _token_ids(case["rows"], case["vocab"], gen)
    elif case["op"] == "embed_grad":
        s["dout"] = (torch.randn(case["rows"], case["width"], generator=gen, device="cuda") * 1e-2).to(DTYPES[case["dtype"]])
        s["ids"] = _token_ids(case["rows"], case["vocab"], gen)
        s["dweight"] = torch.empty(case["vocab"], case["width"], device="cuda")
        if case["accumulate"]:
            s["dweight"].normal_(0, 1e-2, generator=gen)
    else:
        sizes = _sizes(case)

        def normal(std):
            return lambda n: torch.randn(n, generator=gen, device="cuda") * std

        s["p"] = _flat(sizes, normal(0.02))
        s["g"] = _flat(sizes, normal(1e-2)).to(DTYPES[case["dtype"]])
        m = _flat(sizes, normal(1e-3))
        v = _flat(sizes, lambda n: torch.rand(n, generator=gen, device="cuda") * 1e-4)
        if case["bits"] == 8:
            s["m"], s["ms"] = _to_codes(m, False)
            s["v"], s["vs"] = _to_codes(v.sqrt(), True)
        else:
            s["m"], s["v"] = m, v
        if case["copy"]:
            s["low"] = torch.zeros(s["p"].numel(), dtype=torch.bfloat16, device="cuda")
    if own:
        _handles(case, s)
    return s


# ---- the framework's calls -----------------------------------------------------

def _handles(case, s):
    """The framework's tensors over the same memory, and the outputs that a training loop keeps."""
    import rusttorch_b200 as rt

    names = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.float16: "float16", torch.int64: "int64",
             torch.float8_e4m3fn: "float8_e4m3"}

    def wrap(t, shape=None):
        return rt.Tensor.from_device_ptr(t.data_ptr(), list(t.shape) if shape is None else shape, owner=t, dtype=names[t.dtype])

    h = {"rt": rt}
    if case["op"] in ("loss_grad", "loss_tape"):
        s["loss"] = torch.empty(1, device="cuda")
        s["dlogits"] = torch.empty_like(s["logits"])
        for k in ("logits", "targets", "loss", "dlogits"):
            h[k] = wrap(s[k])
        if case["op"] == "loss_tape":
            s["stats"] = torch.empty(case["rows"], 3, device="cuda")
            h["stats"], h["upstream"] = wrap(s["stats"]), wrap(s["upstream"])
    elif case["op"] == "embed":
        s["out"] = torch.empty(case["rows"], case["width"], dtype=s["weight"].dtype, device="cuda")
        for k in ("weight", "ids", "out"):
            h[k] = wrap(s[k])
    elif case["op"] == "embed_grad":
        for k in ("dout", "ids", "dweight"):
            h[k] = wrap(s[k])
    else:
        sizes = _sizes(case)
        starts, blocks, _ = _layout(sizes)
        for k in ("p", "g", "m", "v", "low"):
            h[k] = rt.TensorList([wrap(s[k][a:a + n]) for a, n in zip(starts, sizes)]) if k in s else None
        for k in ("ms", "vs"):
            h[k] = rt.TensorList([wrap(s[k][a // BLOCK:a // BLOCK + n]) for a, n in zip(starts, blocks)]) if k in s else None
    s["own"] = h


def _run_own(s):
    h = s["own"]
    rt = h["rt"]
    if s["op"] == "loss_grad":
        rt.softmax_cross_entropy_grad(h["logits"], h["targets"], ignore_index=IGNORE, loss=h["loss"], grad=h["dlogits"])
        return {"loss": s["loss"], "dlogits": s["dlogits"]}
    if s["op"] == "loss_tape":
        rt.softmax_cross_entropy(h["logits"], h["targets"], ignore_index=IGNORE, loss=h["loss"], stats=h["stats"])
        rt.softmax_cross_entropy_backward(h["upstream"], h["logits"], h["targets"], h["stats"], ignore_index=IGNORE, out=h["dlogits"])
        return {"loss": s["loss"], "dlogits": s["dlogits"]}
    if s["op"] == "embed":
        rt.embedding(h["weight"], h["ids"], scale=math.sqrt(s["width"]), out=h["out"])
        return {"out": s["out"]}
    if s["op"] == "embed_grad":
        rt.embedding_backward(h["dout"], h["ids"], s["vocab"], scale=math.sqrt(s["width"]), padding_idx=0,
                              accumulate=s["accumulate"], out=h["dweight"])
        return {"dweight": s["dweight"]}
    rt.adamw_update_multi(h["p"], h["g"], h["m"], h["v"], LR, B1, B2, EPS, WD, STEP, m_scales=h["ms"], v_scales=h["vs"],
                          copies=h["low"], seed=STEP)
    return _adamw_outputs(s)


# ---- the plain forms -----------------------------------------------------------

def _plain_loss(s, upstream):
    """loss = mean over the counted rows of log(sum_j e^(x_j - x_t)); its gradient (softmax - onehot) / count."""
    logits, targets = s["logits"], s["targets"]
    counted = targets != IGNORE
    t = torch.where(counted, targets, 0)[:, None]
    count = counted.sum().clamp(min=1)
    x = logits.float()
    top = x.amax(1, keepdim=True)
    xt = x.gather(1, t)
    e = (x - top).exp_()
    et = e.gather(1, t)
    others = e.scatter(1, t, 0.0).sum(1, keepdim=True)      # a sum next to 1 keeps its digits without the target's term
    total = others + et
    row = torch.where(xt == top, torch.log1p(others), total.log() - (xt - top))
    loss = torch.where(counted, row[:, 0], 0.0).double().sum() / count
    factor = torch.where(counted, upstream / count, torch.zeros_like(upstream))[:, None]
    grad = e.div_(total).scatter_(1, t, -others / total).mul_(factor)
    grad = torch.where(counted[:, None], grad, 0.0)
    return {"loss": loss.float().reshape(1), "dlogits": grad.to(logits.dtype)}


def _mix(x):
    """32 random bits of each counter, in the low half of an int64."""
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _key(seed, i):
    """The low 32 bits of splitmix64's element i: one tensor's key."""
    m = (1 << 64) - 1
    z = (seed + (i + 1) * 0x9E3779B97F4A7C15) & m
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & m
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & m
    return (z ^ (z >> 31)) & 0xFFFFFFFF


def _scale(top):
    """The least power of two that brings `top` to 448 or below, not under 2^-126."""
    f, k = torch.frexp(top)
    e = torch.where(top > 0, k.int() - 9 + (f > 0.875).int(), -126).clamp(min=-126)
    return ((e + 127) << 23).view(torch.float32)


def _encode(x, bits16, least):
    """x [blocks, BLOCK] in e4m3 under each block's power of two, rounded up with the probability of what is cut off."""
    size = x.abs()
    scale = _scale(torch.where(torch.isfinite(size), size, 0.0).amax(1))
    y = size / scale[:, None]
    low = y < 2.0 ** -6
    z = torch.where(low, y + 2.0 ** -6, y)
    z = ((z.view(torch.int32) + ((bits16 << 4) + 8).int()) & -(1 << 20)).view(torch.float32)
    z = torch.where(low, z - 2.0 ** -6, z)
    if least:
        z = torch.where((y > 0) & (z == 0), 2.0 ** -9, z)
    z = torch.where(torch.isfinite(size), z, math.nan)
    return torch.copysign(z, x).to(torch.float8_e4m3fn), scale


def _plain_adamw(s):
    b1, b2 = np.float32(B1), np.float32(B2)
    omb1, omb2 = float(np.float32(1) - b1), float(np.float32(1) - b2)
    b1, b2 = float(b1), float(b2)
    bc1, bc2 = 1 - B1 ** STEP, 1 - B2 ** STEP
    p, g = s["p"], s["g"].float()
    decay = p * float(np.float32(LR * WD))
    if s["bits"] == 32:
        m = s["m"].mul_(b1).add_(g * omb1)
        v = s["v"].mul_(b2).add_((g * g).mul_(omb2))
        den = (v / float(np.float32(bc2))).sqrt_().add_(EPS)
        p.sub_((m / float(np.float32(bc1))).div_(den).mul_(LR)).sub_(decay)
    else:
        m = (s["m"].float().view(-1, BLOCK) * s["ms"][:, None])
        root = (s["v"].float().view(-1, BLOCK) * s["vs"][:, None])
        g = g.view(-1, BLOCK)
        m = m.mul_(b1).add_(g * omb1)
        root = (root * root).mul_(b2).add_((g * g).mul_(omb2)).sqrt_()
        den = (root * float(np.float32(1 / math.sqrt(bc2)))).add_(EPS)
        p.sub_((m / den).mul_(float(np.float32(LR / bc1))).view(-1)).sub_(decay)
        sizes = _sizes(s)
        tensor, start = _blocks(sizes)
        key = torch.tensor([_key(STEP, i) for i in range(len(sizes))], dtype=torch.int64).cuda()[tensor]
        inside = start[:, None] + torch.arange(BLOCK, device="cuda")
        bits = _mix(key[:, None] + (inside & 0xFFFFFFFF) * 0x9E3779B1 + (inside >> 32) * 0xBB67AE85)
        c, scale = _encode(m, bits & 0xFFFF, False)
        s["m"].copy_(c.view(-1))
        s["ms"].copy_(scale)
        c, scale = _encode(root, bits >> 16, True)
        s["v"].copy_(c.view(-1))
        s["vs"].copy_(scale)
    if "low" in s:
        s["low"].copy_(p)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {k: s[k] for k in ("p", "m", "v", "ms", "vs", "low") if k in s}


def run(state):
    if own:
        return _run_own(state)
    s = state
    if s["op"] == "loss_grad":
        return _plain_loss(s, torch.ones(1, device="cuda"))
    if s["op"] == "loss_tape":
        return _plain_loss(s, s["upstream"])
    if s["op"] == "embed":
        return {"out": (s["weight"][s["ids"]].float() * math.sqrt(s["width"])).to(s["weight"].dtype)}
    if s["op"] == "embed_grad":
        total = torch.zeros(s["vocab"], s["width"], device="cuda").index_add_(0, s["ids"], s["dout"].float())
        total[0] = 0
        total.mul_(math.sqrt(s["width"]))
        if s["accumulate"]:
            s["dweight"].add_(total)
        else:
            s["dweight"].copy_(total)
        return {"dweight": s["dweight"]}
    return _plain_adamw(s)


def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] in ("loss_grad", "loss_tape"):
        cells = case["rows"] * case["vocab"]
        return {"bytes": 2 * cells * size + 8 * case["rows"], "flops": 6 * cells}
    if case["op"] in ("embed", "embed_grad"):
        n, d, v = case["rows"], case["width"], case["vocab"]
        kinds = _distinct(n, v)
        if case["op"] == "embed":
            return {"bytes": (kinds + n) * d * size + 8 * n, "flops": n * d}
        rows = 2 * kinds if case["accumulate"] else v
        return {"bytes": n * d * size + rows * d * 4 + 8 * n, "flops": n * d}
    n = float(sum(_sizes(case)))
    each = 8 + size + (16 if case["bits"] == 32 else 4 + 16 / BLOCK) + (2 if case["copy"] else 0)
    return {"bytes": n * each, "flops": n * 14}


# ---- the definitions in 64 bits --------------------------------------------------

def exact(case, seed):
    s = _bare(case, seed)
    op = case["op"]
    if op in ("loss_grad", "loss_tape"):
        return _exact_loss(s)
    if op == "embed":
        scale = float(np.float32(math.sqrt(case["width"])))
        return {"out": s["weight"].double().index_select(0, s["ids"]) * scale}
    if op == "embed_grad":
        scale = float(np.float32(math.sqrt(case["width"])))
        use = s["ids"] != 0
        total = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        total.index_put_((s["ids"][use],), s["dout"].double()[use], accumulate=True)
        total *= scale
        return {"dweight": total + s["dweight"].double() if case["accumulate"] else total}
    return _exact_adamw(case, s)


def _bare(case, seed):
    """prepare()'s inputs without the framework's tensors."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _exact_loss(s):
    n = s["rows"]
    up = float(s["upstream"][0]) if "upstream" in s else 1.0
    count = max(1, int((s["targets"] != IGNORE).sum()))
    grad = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    loss = 0.0
    for a in range(0, n, 512):
        t = s["targets"][a:a + 512]
        keep = (t != IGNORE).nonzero()[:, 0]
        if not keep.numel():
            continue
        t, x = t[keep], s["logits"][a:a + 512][keep].double()
        at = torch.arange(len(t), device="cuda")
        x -= x[at, t][:, None].clone()              # against the target: its own term is 1
        top = x.amax(1, keepdim=True).clamp(min=0)
        e = torch.exp(x - top)
        one = e[at, t].clone()
        e[at, t] = 0
        rest = e.sum(1)
        big = rest / one
        loss += float(torch.where(one > 0, torch.log1p(big), rest.log() + top[:, 0]).sum())
        part = e / (rest + one)[:, None]
        part[at, t] = -rest / (rest + one)
        grad[a + keep] = part * (up / count)
    return {"loss": torch.tensor([loss / count], dtype=torch.float64), "dlogits": grad}


def _exact_adamw(case, s):
    b1, b2, lr = (float(np.float32(x)) for x in (B1, B2, LR))
    c1, c2 = 1 - B1 ** STEP, 1 - B2 ** STEP
    g, p = s["g"].double(), s["p"].double()
    m, v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        m = (m.view(-1, BLOCK) * s["ms"].double()[:, None]).view(-1)
        v = (v.view(-1, BLOCK) * s["vs"].double()[:, None]).view(-1) ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = p - lr * (m / c1) / ((v / c2).sqrt() + float(np.float32(EPS))) - p * float(np.float32(LR * WD))
    r = {"p": p, "m": m, "v": v}
    if case["bits"] == 8:
        # what the codes stand for before they are rounded; the powers of two have no other value
        for k, x in (("m", m.view(-1, BLOCK)), ("v", v.sqrt().view(-1, BLOCK))):
            top = x.abs().amax(1, keepdim=True).clamp(min=2.0 ** -140)
            e = torch.ceil(torch.log2(top / 448)).clamp(min=-126)
            r[k] = (x * torch.exp2(-e)).view(-1)
        r["ms"] = r["vs"] = None
    if case["copy"]:
        r["low"] = p
    return r
