"""What is timed of the operators of a dense stack that perf/operators.py does
not have: layer norm forward and backward, rows in microscaled 4-bit floating
point with the dense layer that multiplies them, and the update of a weight
made orthogonal by Newton-Schulz products.

Kinds of case
  norm        layer norm of hidden states
  norm-train  the same forward and backward: the output and the gradients of
              the input, the scale and the shift
  mx4-rows    rows quantised to 4-bit codes with a power of two for each 32
              values, and read back
  mx4         a dense layer on such a weight: its input is quantised the same
              way, then product, bias, activation, residual, and for the layer
              that ends in the embedding the division by its length
  update      a gradient made orthogonal
  step        a training step of a weight: momentum, the orthogonal update,
              the weight and its rounded copy

Hidden states have channels of different means and sizes, a few of them large,
as a language model's have; gradients are sums of few strong directions and
noise, as a batch leaves them.
"""
import math

import torch

#: Set by what imports this file: plain torch operations (False) or the
#: framework's operators (True).
own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
BLOCK = 32  # values of a power of two
STEPS, COEFFICIENTS = 5, (3.4445, -4.7750, 2.0315)
RATE, MU, DECAY = 0.02, 0.95, 0.0002


# ---- the cases -----------------------------------------------------------------


def _norm(name, rows, n, type, kind="norm", pad=0, out=None):
    return {"name": name, "kind": kind, "rows": rows, "n": n, "type": type, "out": out or type, "pad": pad}


def _mx4(name, rows, k, n, type, act="none", bias=False, residual=False, normalize=False, out=None, pad=0):
    return {"name": name, "kind": "mx4", "rows": rows, "k": k, "n": n, "type": type, "out": out or type, "act": act,
            "bias": bias, "residual": residual, "normalize": normalize, "pad": pad}


def listed():
    return [
        # one query's 32 tokens between two layers: latency
        _norm("norm-query", 32, 768, "bf16"),
        # a corpus's batch of documents
        _norm("norm-documents", 65_536, 1024, "bf16"),
        # a training step of a batch of documents
        _norm("norm-train", 16_384, 1024, "bf16", kind="norm-train"),
        # 32 queries and their documents in 32 bits, at a width and in rows
        # that fill nothing
        _norm("norm-train-ragged", 6_001, 777, "f32", kind="norm-train", pad=3),
        # the weight of a widening layer, as a program quantises it once
        {"name": "mx4-weight", "kind": "mx4-rows", "rows": 4096, "n": 1024, "type": "f32", "pad": 0},
        # one query of 32 tokens through the layer that ends in its embeddings
        _mx4("mx4-query", 32, 768, 128, "bf16", normalize=True, out="f32"),
        # one token through a widening layer: the weight is read once
        _mx4("mx4-token", 1, 1024, 4096, "f16", act="gelu", bias=True),
        # a corpus's batch of documents through a widening layer
        _mx4("mx4-documents", 65_536, 1024, 4096, "bf16", act="gelu", bias=True),
        # sizes that fill no tile, rows apart from each other, a residual
        _mx4("mx4-ragged", 10_007, 777, 520, "bf16", act="silu", bias=True, residual=True, pad=3),
        # the layer that ends in the embedding, trained in 32 bits
        {"name": "step-embedding", "kind": "step", "rows": 128, "n": 768, "type": "f32", "pad": 0},
        # a layer of a stack, trained in 16 bits
        {"name": "update-square", "kind": "update", "rows": 1024, "n": 1024, "type": "bf16", "pad": 0},
        # a widening layer, trained in 32 bits
        {"name": "step-widening", "kind": "step", "rows": 4096, "n": 1024, "type": "f32", "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm"] * 2 + ["norm-train"] * 3 + ["mx4-rows"] + ["mx4"] * 4 + ["update"] * 2 + ["step"] * 2)
    type = rng.choice(["bf16", "bf16", "f16", "f32"])
    pad = rng.choice([0, 0, 8, 5])
    if kind in ("norm", "norm-train", "mx4-rows"):
        n = _log_int(rng, 48, 8192)
        if rng.random() < 0.6:
            n = -(-n // 64) * 64
        most = {"norm": 2**26, "norm-train": 2**24, "mx4-rows": 2**22}[kind]
        rows = _log_int(rng, 1, min(65_536, most // n))
        case = {"kind": kind, "rows": rows, "n": n, "type": type, "pad": pad}
        return case if kind == "mx4-rows" else {**case, "out": "f32" if rng.random() < 0.2 else type}
    if kind == "mx4":
        normalize = rng.random() < 0.4
        n = rng.choice([128, 128, 96, 64, 48]) if normalize else _log_int(rng, 64, 4096)
        k = _log_int(rng, 128, 4096)
        if rng.random() < 0.7:
            n, k = (n if normalize else -(-n // 64) * 64), -(-k // 64) * 64
        rows = _log_int(rng, 1, max(2, min(65_536, 2**38 // (n * k), 2**28 // (n + k))))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "type": type,
                "out": "f32" if normalize and rng.random() < 0.5 else type,
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.4, "normalize": normalize, "pad": pad}
    rows, n = _log_int(rng, 48, 4096), _log_int(rng, 48, 4096)
    if rng.random() < 0.6:
        rows, n = -(-rows // 64) * 64, -(-n // 64) * 64
    if min(rows, n) > 1024:  # no more products than the largest listed case
        rows, n = (min(rows, 1408), min(n, 1408))
    return {"kind": kind, "rows": rows, "n": n, "type": type, "pad": pad}


# ---- inputs --------------------------------------------------------------------


def _rows(gen, rows, n, type, pad):
    """Hidden states [rows, n], `pad` values apart from each other."""
    wide = n + pad
    x = torch.randn(rows, wide, generator=gen, device="cuda")
    size = torch.exp(0.5 * torch.randn(wide, generator=gen, device="cuda"))
    size[torch.randint(0, wide, (1 + wide // 256,), generator=gen, device="cuda")] *= 8.0
    x.mul_(size).add_(0.3 * size * torch.randn(wide, generator=gen, device="cuda"))
    return x.to(TYPES[type])[:, :n]


def _apart(rows, n, type, pad):
    return torch.zeros(rows, n + pad, dtype=TYPES[type], device="cuda")[:, :n]


def _prepare_norm(case, gen):
    rows, n, type, out, pad = case["rows"], case["n"], case["type"], case["out"], case["pad"]
    t = {"x": _rows(gen, rows, n, type, pad),
         "weight": (1.0 + 0.2 * torch.randn(n, generator=gen, device="cuda")).to(TYPES[type]),
         "bias": (0.1 * torch.randn(n, generator=gen, device="cuda")).to(TYPES[type]),
         "y": _apart(rows, n, out, pad)}
    if case["kind"] == "norm-train":
        t["dy"] = torch.randn(rows, n + pad, generator=gen, device="cuda").to(TYPES[out])[:, :n]
        # what the forward pass keeps for the backward pass, and the gradients
        t["mean"], t["rstd"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        t["dx"] = _apart(rows, n, type, pad)
        t["dweight"], t["dbias"] = torch.empty_like(t["weight"]), torch.empty_like(t["bias"])
    return t


def _power(e):
    """2^e in 32 bits for whole numbers of -127 to 127."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantise(x):
    """Rows [m, n] as 4-bit values and exponents: [m, blocks, 32] of 0, 0.5, 1,
    1.5, 2, 3, 4 and 6 with their signs, and [m, blocks] whole numbers e with
    row = value 2^e. e is the exponent of a block's largest magnitude less 2,
    at least -127."""
    m, n = x.shape
    blocks = -(-n // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - n)).view(m, blocks, BLOCK)
    most = x.abs().amax(2)
    e = torch.where(most > 0, (torch.frexp(most).exponent - 3).clamp(min=-127), -127)
    v = x / _power(e).unsqueeze(2)
    size = v.abs()
    # steps of 1/2 up to 2, of 1 up to 4, of 2 above; ties to the even code
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    return torch.copysign((torch.round(size / step) * step).clamp(max=6.0), v), e


def _pack(values, e):
    """Codes [m, 16 blocks] uint8, the even value in the low half of a byte,
    and scales [m, blocks rounded up to 8] uint8: e + 127."""
    size = values.abs()
    code = (2 * size - (size - 2).clamp(min=0) - 0.5 * (size - 4).clamp(min=0)).to(torch.uint8)
    code = code | (torch.signbit(values).to(torch.uint8) << 3)
    code = code.flatten(1)
    scales = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -e.shape[1] % 8))
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scales.contiguous()


def _unpack(codes, scales, n):
    """The rows [m, n] that codes and scales stand for, in 32 bits."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :n]
    size = (c & 7).float()
    size = 0.5 * (size + (size - 4).clamp(min=0)) + (size - 6).clamp(min=0)
    power = _power(scales.to(torch.int32) - 127).repeat_interleave(BLOCK, 1)[:, :n]
    return torch.where(c >= 8, -size, size) * power


def _prepare_rows(case, gen):
    rows, n = case["rows"], case["n"]
    blocks = -(-n // BLOCK)
    return {"x": _rows(gen, rows, n, case["type"], case["pad"]), "out": _apart(rows, n, case["type"], case["pad"]),
            "codes": torch.zeros(rows, 16 * blocks, dtype=torch.uint8, device="cuda"),
            "scales": torch.zeros(rows, -(-blocks // 8) * 8, dtype=torch.uint8, device="cuda")}


def _prepare_mx4(case, gen):
    rows, k, n, type = case["rows"], case["k"], case["n"], case["type"]
    codes, scales = _pack(*_quantise(torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)))
    return {"x": _rows(gen, rows, k, type, case["pad"]), "codes": codes, "scales": scales,
            "bias": (0.1 * torch.randn(n, generator=gen, device="cuda")).to(TYPES[type]) if case["bias"] else None,
            "residual": torch.randn(rows, n + case["pad"], generator=gen, device="cuda").to(TYPES[type])[:, :n]
            if case["residual"] else None,
            "y": _apart(rows, n, case["out"], case["pad"])}


def _gradient(gen, rows, n, type, pad):
    few = max(1, min(rows, n) // 8)
    strong = torch.randn(rows, few, generator=gen, device="cuda") @ torch.randn(few, n, generator=gen, device="cuda")
    g = torch.zeros(rows, n + pad, device="cuda")
    g[:, :n] = 1e-3 * (strong / math.sqrt(few) + 0.3 * torch.randn(rows, n, generator=gen, device="cuda"))
    return g.to(TYPES[type])[:, :n]


def _prepare_update(case, gen):
    rows, n, type = case["rows"], case["n"], case["type"]
    t = {"gradient": _gradient(gen, rows, n, type, case["pad"])}
    if case["kind"] == "update":
        return {**t, "out": _apart(rows, n, type, case["pad"])}
    t["weight"] = torch.randn(rows, n, generator=gen, device="cuda") / math.sqrt(n)
    t["momentum"] = 5.0 * _gradient(gen, rows, n, "f32", 0).contiguous()
    # the next step's, so that a step can be made again
    t["new_weight"], t["new_momentum"] = torch.empty_like(t["weight"]), torch.empty_like(t["momentum"])
    t["rounded"] = _apart(rows, n, type, case["pad"]) if type != "f32" else None
    return t


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind in ("norm", "norm-train"):
        t = _prepare_norm(case, gen)
    elif kind == "mx4-rows":
        t = _prepare_rows(case, gen)
    elif kind == "mx4":
        t = _prepare_mx4(case, gen)
    else:
        t = _prepare_update(case, gen)
    return {"case": case, "t": t}


# ---- the plain forms -----------------------------------------------------------


def _plain_norm(t, case):
    x, w = t["x"].float(), t["weight"].float()
    d = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    unit = d * rstd
    y = (unit * w + t["bias"].float()).to(TYPES[case["out"]])
    if case["kind"] == "norm":
        return y
    dy = t["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    type = TYPES[case["type"]]
    return {"y": y, "dx": dx.to(type), "dweight": (dy * unit).sum(0).to(type), "dbias": dy.sum(0).to(type)}


def _plain_rows(t, case):
    values, e = _quantise(t["x"])
    return (values * _power(e).unsqueeze(2)).flatten(1)[:, :case["n"]].to(TYPES[case["type"]])


def _activation(z, act):
    if act == "relu":
        return z.clamp(min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain_mx4(t, case):
    values, e = _quantise(t["x"])
    x = (values * _power(e).unsqueeze(2)).flatten(1)[:, :case["k"]]
    z = x @ _unpack(t["codes"], t["scales"], case["k"]).t()
    if case["bias"]:
        z = z + t["bias"].float()
    h = _activation(z, case["act"])
    if case["residual"]:
        h = h + t["residual"].float()
    if case["normalize"]:
        h = h / h.norm(dim=1, keepdim=True).clamp(min=1e-12)
    return h.to(TYPES[case["out"]])


def _newton_schulz(u):
    """u [m, n] over its norm, then X <- a X + (b A + c A^2) X with A = X X^T,
    on the side with fewer rows."""
    a, b, c = COEFFICIENTS
    x = u if u.shape[0] <= u.shape[1] else u.t()
    # a size's error grows with the singular values
    x = (x.double() / x.double().norm()).float()
    for _ in range(STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x if u.shape[0] <= u.shape[1] else x.t()


def _plain_update(t, case):
    g = t["gradient"].float()
    if case["kind"] == "update":
        return _newton_schulz(g).to(TYPES[case["type"]])
    momentum = MU * t["momentum"] + g
    weight = (1.0 - DECAY) * t["weight"] - RATE * _newton_schulz(g + MU * momentum)
    out = {"momentum": momentum, "weight": weight}
    return out if t["rounded"] is None else {**out, "rounded": weight.to(TYPES[case["type"]])}


def _plain(state):
    case, t = state["case"], state["t"]
    if case["kind"] in ("norm", "norm-train"):
        return _plain_norm(t, case)
    if case["kind"] == "mx4-rows":
        return _plain_rows(t, case)
    if case["kind"] == "mx4":
        return _plain_mx4(t, case)
    return _plain_update(t, case)


# ---- one pass ------------------------------------------------------------------

_context = None


def _handle(state):
    """What a program keeps beside its data: the context, the arrays and the
    layer or the update that its calls are made on."""
    global _context
    from chimera_amd import capi, operators

    if _context is None:
        _context = capi.Context(None, 1, 1, 1, 1)
    case, t = state["case"], state["t"]
    b = state["b"] = {name: None if v is None else operators.from_torch(v) for name, v in t.items()}
    if case["kind"] in ("norm", "norm-train"):
        return operators.LayerNorm(_context, b["weight"], b["bias"], eps=EPS, max_rows=case["rows"],
                                   training=case["kind"] == "norm-train")
    if case["kind"] == "mx4-rows":
        return operators
    if case["kind"] == "mx4":
        return operators.Mx4Linear(_context, b["codes"], b["scales"], case["k"], b["bias"], type=case["type"],
                                   activation=case["act"], normalize=case["normalize"], max_rows=case["rows"])
    return operators.OrthogonalUpdate(_context, case["rows"], case["n"], type=case["type"], steps=STEPS,
                                      coefficients=COEFFICIENTS)


def _own(state):
    handle = state.get("handle")
    if handle is None:
        handle = state["handle"] = _handle(state)
    case, t, b = state["case"], state["t"], state["b"]
    kind = case["kind"]
    if kind == "norm":
        handle.forward(b["x"], b["y"])
        return t["y"]
    if kind == "norm-train":
        handle.forward(b["x"], b["y"], mean=b["mean"], rstd=b["rstd"])
        handle.backward(b["x"], b["dy"], b["mean"], b["rstd"], dx=b["dx"], dweight=b["dweight"], dbias=b["dbias"])
        return {name: t[name] for name in ("y", "dx", "dweight", "dbias")}
    if kind == "mx4-rows":
        handle.mx4_quantise(_context, b["x"], b["codes"], b["scales"])
        handle.mx4_read(_context, b["codes"], b["scales"], b["out"])
        return t["out"]
    if kind == "mx4":
        handle.forward(b["x"], b["y"], residual=b["residual"])
        return t["y"]
    if kind == "update":
        handle.orthogonalize(b["gradient"], b["out"])
        return t["out"]
    handle.step(b["gradient"], b["weight"], b["new_weight"], rate=RATE, decay=DECAY, momentum=b["momentum"],
                new_momentum=b["new_momentum"], mu=MU, nesterov=True, rounded=b["rounded"])
    out = {"momentum": t["new_momentum"], "weight": t["new_weight"]}
    return out if t["rounded"] is None else {**out, "rounded": t["rounded"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------


def _mx4_bytes(rows, n):
    blocks = -(-n // BLOCK)
    return rows * 17 * blocks


def work(case):
    kind, rows, n, e = case["kind"], case["rows"], case["n"], TYPES[case["type"]].itemsize
    if kind in ("norm", "norm-train"):
        o = TYPES[case["out"]].itemsize
        bytes = rows * n * (e + o) + 2 * n * e
        if kind == "norm":
            return {"bytes": bytes, "flops": 8 * rows * n}
        return {"bytes": bytes + rows * n * (o + e) + 2 * n * e, "flops": 24 * rows * n}
    if kind == "mx4-rows":
        return {"bytes": 2 * (rows * n * e + _mx4_bytes(rows, n)), "flops": 6 * rows * n}
    if kind == "mx4":
        k, o = case["k"], TYPES[case["out"]].itemsize
        return {"bytes": rows * k * e + _mx4_bytes(n, k) + e * (case["bias"] * n + case["residual"] * rows * n) + o * rows * n,
                "flops": 2 * rows * n * k}
    m, k = min(rows, n), max(rows, n)
    bytes = 2 * rows * n * e if kind == "update" else rows * n * (e + 16 + (e if e == 2 else 0))
    # of the products A and A^2 one half: they are symmetric
    return {"bytes": bytes, "flops": STEPS * (3 * m * m * k + m * m * m)}


# ---- the definitions in 64 bits ------------------------------------------------


def _exact_norm(t, case):
    x, w, n = t["x"].double(), t["weight"].double(), case["n"]
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sigma = (var + EPS).sqrt()
    z = (x - mean) / sigma
    y = torch.addcmul(t["bias"].double(), z, w)
    if case["kind"] == "norm":
        return y
    dy = t["dy"].double()
    dz = dy * w
    # the derivative of z by x is (1 - 1 1^T / n - z z^T / n) / sigma
    dx = torch.addcmul(dz - dz.sum(1, keepdim=True) / n, z, torch.linalg.vecdot(z, dz).unsqueeze(1) / n, value=-1) / sigma
    return {"y": y, "dx": dx, "dweight": torch.linalg.vecdot(dy, z, dim=0), "dbias": dy.sum(0)}


def _exact_blocks(x):
    """Rows in 64 bits as 4-bit values times their powers of two, by the
    nearest of the 15 values (the even code where two are as near)."""
    n = x.shape[1]
    x = x.double()
    rows = torch.empty_like(x)
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    for at in range(0, n, BLOCK):
        part = x[:, at:at + BLOCK]
        most = part.abs().amax(1, keepdim=True)
        power = torch.exp2(torch.floor(torch.log2(most.clamp(min=2.0**-200))) - 2).clamp(min=2.0**-127)
        size = part.abs() / power
        best = torch.zeros_like(size)
        for i in range(1, 8):
            border = (levels[i - 1] + levels[i]) / 2
            best = torch.where((size > border) | ((size == border) & (i % 2 == 0)), levels[i], best)
        rows[:, at:at + BLOCK] = torch.sign(part) * best * power
    return rows


def _exact_mx4(t, case):
    k = case["k"]
    codes = t["codes"].long()
    at = torch.arange(k, device=codes.device)
    c = (codes[:, at // 2] >> (4 * (at % 2))) & 15
    exponent, mantissa = (c >> 1) & 3, (c & 1).double()
    w = torch.where(exponent > 0, (1 + mantissa / 2) * torch.exp2((exponent - 1).double()), mantissa / 2)
    w = torch.where(c >= 8, -w, w) * torch.exp2(t["scales"].double() - 127)[:, at // BLOCK]
    z = _exact_blocks(t["x"]) @ w.T.contiguous()
    if case["bias"]:
        z += t["bias"].double()
    if case["act"] == "relu":
        z = torch.where(z > 0, z, 0.0)
    elif case["act"] == "gelu":
        z = z * torch.special.erfc(-z / math.sqrt(2)) / 2
    elif case["act"] == "gelu_tanh":
        z = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z**3))
    elif case["act"] == "silu":
        z = z * torch.sigmoid(z)
    if case["residual"]:
        z += t["residual"].double()
    if case["normalize"]:
        z /= z.square().sum(1, keepdim=True).sqrt().clamp(min=1e-12)
    return z


def _exact_orthogonal(u):
    """By the eigenvalues of U U^T: the products are a polynomial of them."""
    wide = u.shape[0] <= u.shape[1]
    x = u if wide else u.T
    x = x / x.square().sum().sqrt()
    values, vectors = torch.linalg.eigh((x @ x.T.contiguous()).cpu())
    a, b, c = COEFFICIENTS
    total = torch.ones_like(values)
    for _ in range(STEPS):
        square = values * total * total
        total = total * (a + b * square + c * square * square)
    vectors, total = vectors.cuda(), total.cuda()
    x = (vectors * total) @ (vectors.T.contiguous() @ x.contiguous())
    return x if wide else x.T


def exact(case, seed):
    t = prepare(case, seed)["t"]
    kind = case["kind"]
    if kind in ("norm", "norm-train"):
        return _exact_norm(t, case)
    if kind == "mx4-rows":
        return _exact_blocks(t["x"])
    if kind == "mx4":
        return _exact_mx4(t, case)
    g = t["gradient"].double()
    if kind == "update":
        return _exact_orthogonal(g)
    momentum = MU * t["momentum"].double() + g
    weight = (1 - DECAY) * t["weight"].double() - RATE * _exact_orthogonal(g + MU * momentum)
    out = {"momentum": momentum, "weight": weight}
    return out if t["rounded"] is None else {**out, "rounded": weight}
