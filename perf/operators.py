"""What is timed of the token operators: the dense layers that turn a
language model's hidden states into token embeddings, forward and backward,
the quantised cache that the embeddings of changing documents are written to
and read back from, and late interaction (MaxSim) on that cache.

Kinds of case
  dense   one dense layer: product, bias, activation, residual, and for the
          layer that ends in the embedding the division by its length
  train   the same layer forward and backward: the output and the gradients
          of the input, the weight, the bias and the residual
  store   embeddings written to the slots of a cache and read back
  read    tokens of documents in the order of a candidate list, read back
  maxsim  the sum over a query's tokens of the best product with a
          document's cached tokens, for every candidate of every query

Hidden states are normal, weights keep their scale, embeddings are Gaussian
mixtures on the unit sphere and document lengths uniform or clipped
log-normal, as in the repository's benchmark configurations. Pages of a cache
are in no order, as after documents came and went.
"""
import math

import numpy as np
import torch

#: Set by what imports this file: plain torch operations (False) or the
#: framework's operators (True).
own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LARGEST_CODE = {"int8": 127.0, "int4": 7.0, "fp8": 448.0}
BITS = {"int8": 8, "int4": 4, "fp8": 8}


# ---- the cases -----------------------------------------------------------------


def _dense(name, rows, k, n, type, act="none", bias=False, residual=False, normalize=False, out=None, pad=0,
           kind="dense"):
    return {"name": name, "kind": kind, "rows": rows, "k": k, "n": n, "type": type, "out": out or type, "act": act,
            "bias": bias, "residual": residual, "normalize": normalize, "pad": pad}


def _maxsim(name, nq, q_len, type, format, docs, lens, longest, cands, dim=128, group=128, page=16):
    return {"name": name, "kind": "maxsim", "nq": nq, "q_len": q_len, "type": type, "format": format, "docs": docs,
            "lens": lens, "longest": longest, "cands": cands, "dim": dim, "group": group, "page": page}


def listed():
    return [
        # one query of 32 tokens through the layer that ends in its
        # embeddings: the latency of a served query
        _dense("dense-query", 32, 768, 128, "bf16", normalize=True, out="f32"),
        # one token through a widening layer: the weight is read once
        _dense("dense-token", 1, 1024, 4096, "f16", act="gelu", bias=True),
        # a corpus's batch of documents through a widening layer
        _dense("dense-documents", 65_536, 1024, 4096, "bf16", act="gelu", bias=True),
        # sizes that fill no tile, rows apart from each other, a residual
        _dense("dense-ragged", 10_007, 777, 520, "bf16", act="silu", bias=True, residual=True, pad=3),
        # an encoder that runs in 32 bits: documents into embeddings
        _dense("dense-f32", 20_000, 768, 96, "f32", normalize=True),
        # a training step of a layer of a dense stack
        _dense("train-residual", 16_384, 1024, 1024, "bf16", act="gelu", bias=True, residual=True, kind="train"),
        # a training step of the last layer: 32 queries and their documents
        _dense("train-embedding", 6_001, 768, 128, "f32", bias=True, normalize=True, kind="train"),
        # one document's tokens as they are added
        {"name": "store-document", "kind": "store", "rows": 180, "slots": 65_536, "type": "f32", "format": "int8",
         "dim": 128, "group": 128},
        # a corpus of 2M tokens written, from an encoder's 16-bit output
        {"name": "store-corpus", "kind": "store", "rows": 2_000_000, "slots": 2_400_000, "type": "bf16",
         "format": "int4", "dim": 128, "group": 32},
        # one query's 100 candidates on the cache: latency
        _maxsim("maxsim-query", 1, 32, "f32", "int8", 20_000, "lognormal", 300, 100),
        # the rescoring configuration: 256 queries of 300 candidates
        _maxsim("maxsim-batch", 256, 32, "f32", "int8", 100_000, "uniform", 256, 300),
        # two queries of odd length on a few long documents, 4-bit codes
        _maxsim("maxsim-long", 2, 19, "bf16", "int4", 8, "ragged", 60_000, 4, dim=96, group=32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["dense"] * 4 + ["train"] * 2 + ["store", "store", "read"] + ["maxsim"] * 4)
    if kind in ("dense", "train"):
        type = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
        normalize = rng.random() < 0.4
        n = rng.choice([128, 128, 96, 64, 48]) if normalize else _log_int(rng, 64, 4096)
        k = _log_int(rng, 128, 4096)
        if rng.random() < 0.7:
            n, k = (n if normalize else -(-n // 64) * 64), -(-k // 64) * 64
        most = {"dense": 2**38, "train": 2**36}[kind] // (8 if type == "f32" else 1)
        rows = _log_int(rng, 1, max(2, min(65_536, most // (n * k), 2**28 // (n + k))))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "type": type,
                "out": "f32" if normalize and rng.random() < 0.5 else type,
                # no relu: at its kink the last bit of a sum decides the derivative
                "act": rng.choice(["none", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.4, "normalize": normalize, "pad": rng.choice([0, 0, 8, 5])}
    format = rng.choice(["int8", "int4", "fp8"])
    dim = rng.choice([128, 128, 128, 96, 100, 64, 48])
    group = rng.choice([32, 64, 128])
    if kind in ("store", "read"):
        rows = _log_int(rng, 1, 2_000_000)
        return {"kind": kind, "rows": rows, "slots": 64 + round(rows * rng.uniform(1.0, 1.3)),
                "type": rng.choice(["f32", "bf16", "f16"]), "format": format, "dim": dim, "group": group}
    type = rng.choice(["f32", "f32", "bf16", "f16"])
    page = rng.choice([8, 16, 32, 64])
    q_len = rng.choice([32, 32, 32, rng.randint(1, 31), rng.randint(33, 80)])
    if rng.random() < 0.2:
        docs = rng.randint(2, 12)
        return {"kind": kind, "nq": rng.randint(1, 4), "q_len": q_len, "type": type, "format": format, "docs": docs,
                "lens": "ragged", "longest": _log_int(rng, 2000, 60_000), "cands": rng.randint(1, 4), "dim": dim,
                "group": group, "page": page}
    longest = _log_int(rng, 32, 300)
    cands = _log_int(rng, 10, 300)
    nq = _log_int(rng, 1, max(2, min(256, 15_000_000 // (cands * longest))))
    return {"kind": kind, "nq": nq, "q_len": q_len, "type": type, "format": format,
            "docs": _log_int(rng, 1000, 60_000), "lens": rng.choice(["uniform", "lognormal", "ragged"]),
            "longest": longest, "cands": cands, "dim": dim, "group": group, "page": page}


# ---- inputs --------------------------------------------------------------------


class _Buffer:
    """A torch tensor passed where the operators take device arrays."""

    names = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}

    def __init__(self, tensor):
        self.tensor = tensor
        self.ptr = tensor.data_ptr()
        self.shape = tuple(tensor.shape)
        self.dtype = self.names.get(tensor.dtype, str(tensor.dtype).replace("torch.", ""))
        self.stride = tensor.stride(0) if tensor.dim() == 2 else None


def _buffer(tensor):
    return None if tensor is None else _Buffer(tensor)


def _unit(x):
    return x.div_(x.norm(dim=-1, keepdim=True))


def _tokens(gen, n, dim, centres=4096):
    """n mixture tokens [n, dim]."""
    centre = _unit(torch.randn(centres, dim, generator=gen, device="cuda"))
    out = torch.empty(n, dim, device="cuda")
    for part in out.split(1 << 21):
        label = torch.randint(0, centres, (part.shape[0],), generator=gen, device="cuda")
        torch.randn(part.shape, generator=gen, out=part)
        part.mul_(0.15).add_(centre[label])
        _unit(part)
    return out


def _rows(gen, rows, n, type, pad=0):
    """Normal rows [rows, n], `pad` values apart from each other."""
    return torch.randn(rows, n + pad, generator=gen, device="cuda").to(TYPES[type])[:, :n]


def _prepare_dense(case, gen):
    rows, k, n, type = case["rows"], case["k"], case["n"], case["type"]
    t = {"x": _rows(gen, rows, k, type, case["pad"]),
         "weight": (torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)).to(TYPES[type]),
         "bias": (0.1 * torch.randn(n, generator=gen, device="cuda")).to(TYPES[type]) if case["bias"] else None,
         "residual": _rows(gen, rows, n, type, case["pad"]) if case["residual"] else None,
         "y": torch.empty(rows, n, dtype=TYPES[case["out"]], device="cuda")}
    if case["kind"] == "train":
        t["dy"] = torch.randn(rows, n, generator=gen, device="cuda").to(TYPES[case["out"]])
        # what the forward pass keeps for the backward pass, and the gradients
        t["saved"] = torch.empty(rows, n, dtype=TYPES[type], device="cuda") if case["act"] != "none" else None
        t["norms"] = torch.empty(rows, device="cuda") if case["normalize"] else None
        t["dx"] = torch.empty(rows, k, dtype=TYPES[type], device="cuda")
        t["dweight"] = torch.empty(n, k, dtype=TYPES[type], device="cuda")
        t["dbias"] = torch.empty(n, dtype=TYPES[type], device="cuda") if case["bias"] else None
        t["dresidual"] = (torch.empty(rows, n, dtype=TYPES[type], device="cuda")
                          if case["residual"] and case["normalize"] else None)
    return {"case": case, "t": t, "b": {name: _buffer(v) for name, v in t.items()}}


def _groups(case):
    return -(-case["dim"] // case["group"])


def _row_bytes(case):
    return -(-case["dim"] // 32) * 32 * BITS[case["format"]] // 8


def _quantise(x, format, group):
    """The codes of rows [n, dim] as 32-bit values [n, groups, group], zeros
    after the last value of a row, and one scale a group [n, groups]: the
    largest magnitude over the largest code."""
    n, dim = x.shape
    groups = -(-dim // group)
    x = torch.nn.functional.pad(x.float(), (0, groups * group - dim)).view(n, groups, group)
    most = x.abs().amax(2)
    top = LARGEST_CODE[format]
    inv = torch.where(most > 0, top / most, 0.0)
    scaled = x * inv.unsqueeze(2)
    if format == "fp8":
        codes = scaled.clamp(-top, top).to(torch.float8_e4m3fn).float()
    else:
        codes = scaled.round().clamp(-top, top)
    return codes, most / top


def _pack(codes, case):
    """Codes in the cache's layout [n, row bytes]: rows padded with zeros to a
    multiple of 32 values; 4-bit codes plus 8, the even value in the low bits."""
    n = codes.shape[0]
    wide = -(-case["dim"] // 32) * 32
    codes = torch.nn.functional.pad(codes.reshape(n, -1), (0, 128))[:, :wide]
    if case["format"] == "fp8":
        return codes.to(torch.float8_e4m3fn).view(torch.uint8)
    if case["format"] == "int8":
        return codes.to(torch.int8).view(torch.uint8)
    u = (codes + 8).to(torch.uint8)
    return u[:, 0::2] | (u[:, 1::2] << 4)


def _decode(codes, scales, case):
    """The values [..., dim] in 32 bits of cached rows."""
    if case["format"] == "fp8":
        v = codes.view(torch.float8_e4m3fn).float()
    elif case["format"] == "int8":
        v = codes.view(torch.int8).float()
    else:
        v = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    v = v[..., :case["dim"]]
    return v * scales.repeat_interleave(case["group"], -1)[..., :case["dim"]]


def _filled(gen, slots, case):
    """A cache [slots] of mixture tokens."""
    codes = torch.empty(slots, _row_bytes(case), dtype=torch.uint8, device="cuda")
    scales = torch.empty(slots, _groups(case), device="cuda")
    x = _tokens(gen, slots, case["dim"])
    for at in range(0, slots, 1 << 21):
        part = slice(at, at + (1 << 21))
        c, s = _quantise(x[part], case["format"], case["group"])
        codes[part], scales[part] = _pack(c, case), s
    return codes, scales


def _prepare_store(case, gen):
    rows, slots = case["rows"], case["slots"]
    t = {"slots": torch.randperm(slots, generator=gen, device="cuda")[:rows].contiguous(),
         "out": torch.empty(rows, case["dim"], dtype=TYPES[case["type"]], device="cuda")}
    if case["kind"] == "store":
        t["rows"] = _tokens(gen, rows, case["dim"]).to(TYPES[case["type"]])
        t["codes"] = torch.zeros(slots, _row_bytes(case), dtype=torch.uint8, device="cuda")
        t["scales"] = torch.zeros(slots, _groups(case), device="cuda")
    else:
        t["codes"], t["scales"] = _filled(gen, slots, case)
    return {"case": case, "t": t, "b": {name: _buffer(v) for name, v in t.items()}, "page": 1}


def _doc_lens(rng, case):
    """The quantiles of the length distribution in the seed's order; a
    thirtieth of the documents of a ragged corpus has no token at all."""
    at = (np.arange(case["docs"]) + 0.5) / case["docs"]
    longest = case["longest"]
    if case["lens"] == "uniform":
        low = min(16, longest)
        lens = low + np.floor((longest + 1 - low) * at)
    elif case["lens"] == "lognormal":
        normal = torch.special.ndtri(torch.from_numpy(at)).numpy()
        lens = np.clip(np.rint(np.exp(math.log(longest / 4.5) + 0.5 * normal)), 1, longest)
    else:
        lens = np.maximum(np.floor(longest * (1 - at)) - longest // 30, 0) if longest > 300 else \
            np.maximum(np.floor(longest * at) - longest // 30, 0)
    return rng.permutation(lens.astype(np.int32))


def _prepare_maxsim(case, seed, gen):
    rng = np.random.default_rng(seed)
    lens = _doc_lens(rng, case)
    page = case["page"]
    owned = -(-lens.astype(np.int64) // page)
    start = np.concatenate([[0], np.cumsum(owned)])[:-1]
    pages = int(owned.sum()) + 3
    codes, scales = _filled(gen, pages * page, case)
    order = torch.randperm(pages, generator=gen, device="cuda")[: pages - 3].to(torch.int32)
    nq, q_len = case["nq"], case["q_len"]
    queries = _unit(torch.randn(nq, q_len, case["dim"], generator=gen, device="cuda")).to(TYPES[case["type"]])
    # candidates as a search leaves them: now and then none
    cands = rng.integers(0, case["docs"], size=(nq, case["cands"])).astype(np.int32)
    cands[rng.random(cands.shape) < 0.01] = -1
    # queries of at least half the padded length, the first of all of it
    q_lens = rng.integers((q_len + 1) // 2, q_len + 1, size=nq).astype(np.int32)
    q_lens[0] = q_len
    t = {"codes": codes, "scales": scales, "pages": order, "page_start": torch.from_numpy(start).cuda(),
         "doc_lens": torch.from_numpy(lens).cuda(), "queries": queries, "query_lens": torch.from_numpy(q_lens).cuda(),
         "cands": torch.from_numpy(cands).cuda(), "scores": torch.empty(nq, case["cands"], device="cuda")}
    return {"case": case, "t": t, "b": {name: _buffer(v) for name, v in t.items()}, "page": page,
            "longest": int(lens.max())}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] in ("dense", "train"):
        return _prepare_dense(case, gen)
    if case["kind"] in ("store", "read"):
        return _prepare_store(case, gen)
    return _prepare_maxsim(case, seed, gen)


# ---- the plain forms -----------------------------------------------------------


def _activation(z, act):
    """act(z) and act'(z)."""
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if act == "relu":
        return z.clamp(min=0.0), (z > 0).to(z.dtype)
    return z, None


def _forward(t, case):
    z = t["x"].float() @ t["weight"].float().t()
    if case["bias"]:
        z = z + t["bias"].float()
    h, slope = _activation(z, case["act"])
    if case["residual"]:
        h = h + t["residual"].float()
    if not case["normalize"]:
        return h, slope, None
    norm = h.norm(dim=1, keepdim=True).clamp(min=1e-12)
    return h / norm, slope, norm


def _train(t, case):
    y, slope, norm = _forward(t, case)
    type = TYPES[case["type"]]
    dh = t["dy"].float()
    if case["normalize"]:
        dh = (dh - y * (y * dh).sum(1, keepdim=True)) / norm
    dz = dh if slope is None else dh * slope
    out = {"y": y.to(TYPES[case["out"]]), "dx": (dz @ t["weight"].float()).to(type),
           "dweight": (dz.t() @ t["x"].float()).to(type)}
    if case["bias"]:
        out["dbias"] = dz.sum(0).to(type)
    if t["dresidual"] is not None:
        out["dresidual"] = dh.to(type)
    return out


def _store(t, case):
    codes, scales = _quantise(t["rows"], case["format"], case["group"])
    values = (codes * scales.unsqueeze(2)).flatten(1)[:, :case["dim"]]
    written = torch.zeros_like(t["scales"])
    written[t["slots"]] = scales
    return {"rows": values.to(TYPES[case["type"]]), "scales": written}


def _maxsim_plain(t, case, page, longest):
    nq, cands, dim = case["nq"], case["cands"], case["dim"]
    doc = t["cands"].clamp(min=0).long()
    at = torch.arange(longest, device="cuda")
    lens = torch.where(t["cands"] >= 0, t["doc_lens"][doc], 0)
    valid = at < lens.unsqueeze(2)
    entry = t["page_start"][doc].unsqueeze(2) + at // page
    slot = t["pages"][torch.where(valid, entry, 0)].long() * page + at % page
    slot = slot.flatten(1)
    tokens = _decode(t["codes"][slot], t["scales"][slot], case)
    s = torch.bmm(tokens, t["queries"].float().transpose(1, 2).contiguous())
    s = s.view(nq, cands, longest, -1).masked_fill(~valid.unsqueeze(3), float("-inf")).amax(2)
    real = torch.arange(case["q_len"], device="cuda") < t["query_lens"].unsqueeze(1)
    total = torch.where(real.unsqueeze(1), s, 0.0).sum(2)
    return torch.where(lens > 0, total, float("-inf"))


def _plain(state):
    case, t = state["case"], state["t"]
    if case["kind"] == "dense":
        return _forward(t, case)[0].to(TYPES[case["out"]])
    if case["kind"] == "train":
        return _train(t, case)
    if case["kind"] == "store":
        return _store(t, case)
    if case["kind"] == "read":
        return _decode(t["codes"][t["slots"]], t["scales"][t["slots"]], case).to(TYPES[case["type"]])
    return _maxsim_plain(t, case, state["page"], state["longest"])


# ---- one pass ------------------------------------------------------------------

_context = None


def _handle(state):
    """What a program keeps beside its data: the context, and the layer or
    the cache that its calls are made on."""
    global _context
    from chimera_amd import capi, operators

    if _context is None:
        _context = capi.Context(None, 1, 1, 1, 1)
    case, b = state["case"], state["b"]
    if case["kind"] in ("dense", "train"):
        return operators.Linear(_context, b["weight"], b["bias"], activation=case["act"], normalize=case["normalize"],
                                max_rows=case["rows"], training=case["kind"] == "train")
    return operators.TokenCache(_context, b["codes"], b["scales"], format=case["format"], dim=case["dim"],
                                group=case["group"], page_tokens=state["page"])


def _own(state):
    handle = state.get("handle")
    if handle is None:
        handle = state["handle"] = _handle(state)
    case, t, b = state["case"], state["t"], state["b"]
    if case["kind"] == "dense":
        handle.forward(b["x"], b["y"], residual=b["residual"])
        return t["y"]
    if case["kind"] == "train":
        handle.forward(b["x"], b["y"], residual=b["residual"], saved=b["saved"], norms=b["norms"])
        handle.backward(b["x"], b["dy"], saved=b["saved"], y=b["y"], norms=b["norms"], dx=b["dx"],
                        dweight=b["dweight"], dbias=b["dbias"], dresidual=b["dresidual"])
        out = {"y": t["y"], "dx": t["dx"], "dweight": t["dweight"]}
        if case["bias"]:
            out["dbias"] = t["dbias"]
        if t["dresidual"] is not None:
            out["dresidual"] = t["dresidual"]
        return out
    if case["kind"] == "store":
        handle.write(b["rows"], b["slots"])
        handle.read(b["slots"], b["out"])
        return {"rows": t["out"], "scales": t["scales"]}
    if case["kind"] == "read":
        handle.read(b["slots"], b["out"])
        return t["out"]
    handle.maxsim(b["queries"], b["page_start"], b["doc_lens"], b["pages"], state["longest"], b["cands"], b["scores"],
                  query_lens=b["query_lens"])
    return t["scores"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    if case["kind"] in ("dense", "train"):
        m, k, n = case["rows"], case["k"], case["n"]
        e, o = TYPES[case["type"]].itemsize, TYPES[case["out"]].itemsize
        bytes = e * (m * k + n * k + case["bias"] * n + case["residual"] * m * n) + o * m * n
        if case["kind"] == "dense":
            return {"bytes": bytes, "flops": 2 * m * n * k}
        bytes += o * m * n + e * (m * k + n * k + case["bias"] * n)
        return {"bytes": bytes + (e * m * n if case["residual"] and case["normalize"] else 0), "flops": 6 * m * n * k}
    row = _row_bytes(case) + 4 * _groups(case)
    if case["kind"] in ("store", "read"):
        value = TYPES[case["type"]].itemsize * case["dim"]
        times = 2 if case["kind"] == "store" else 1
        return {"bytes": case["rows"] * times * (row + value + 8), "flops": 4 * case["rows"] * case["dim"]}
    lens = _doc_lens(np.random.default_rng(0), case).astype(np.float64)
    visits = case["nq"] * case["cands"] * float(lens.mean())
    # a token that many candidates share is read once
    tokens = min(visits, float(lens.sum()))
    return {"bytes": tokens * row + case["nq"] * (case["q_len"] * case["dim"] * 4 + case["cands"] * 8),
            "flops": 2 * visits * case["q_len"] * case["dim"]}


# ---- the definitions in 64 bits ------------------------------------------------


def _exact_dense(s, case):
    f = {name: v.double() for name, v in s["t"].items() if v is not None and name in ("x", "weight", "bias", "residual", "dy")}
    pre = torch.matmul(f["x"], f["weight"].T) + f.get("bias", 0.0)
    act, root2 = case["act"], math.sqrt(2.0)
    if act == "gelu":
        cdf = torch.special.erfc(-pre / root2) / 2
        value, slope = pre * cdf, cdf + pre * torch.exp(-pre.square() / 2) / math.sqrt(2 * math.pi)
    elif act == "gelu_tanh":
        # 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u))
        gate = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (pre + 0.044715 * pre**3))
        value = pre * gate
        slope = gate + pre * gate * (1 - gate) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * pre.square())
    elif act == "silu":
        gate = torch.sigmoid(pre)
        value, slope = pre * gate, gate + pre * gate * (1 - gate)
    elif act == "relu":
        value, slope = torch.where(pre > 0, pre, 0.0), torch.where(pre > 0, 1.0, 0.0).double()
    else:
        value, slope = pre, torch.ones_like(pre)
    value = value + f.get("residual", 0.0)
    length = value.square().sum(1).sqrt().clamp(min=1e-12)[:, None] if case["normalize"] else 1.0
    y = value / length
    if case["kind"] == "dense":
        return y
    grad = f["dy"]
    if case["normalize"]:
        grad = (grad - (grad * y).sum(1)[:, None] * y) / length
    inner = grad * slope
    out = {"y": y, "dx": inner @ f["weight"], "dweight": torch.matmul(inner.T, f["x"])}
    if case["bias"]:
        out["dbias"] = inner.sum(0)
    if case["residual"] and case["normalize"]:
        out["dresidual"] = grad
    return out


def _exact_values(codes, scales, case):
    """Cached rows as float64 [n, dim], from the layout's definition."""
    dim, bits = case["dim"], codes.long()
    if case["format"] == "int4":
        col = torch.arange(dim, device=codes.device)
        v = (((bits[:, col // 2] >> (4 * (col % 2))) & 15) - 8).double()
    elif case["format"] == "int8":
        v = (((bits + 128) & 255) - 128).double()[:, :dim]
    else:
        mantissa, exponent = (bits & 7).double(), (bits >> 3) & 15
        v = torch.where(exponent > 0, (8 + mantissa) * torch.pow(2.0, (exponent - 10).double()),
                        mantissa * 2.0**-9)
        v = torch.where(bits >= 128, -v, v)[:, :dim]
    which = torch.arange(dim, device=codes.device) // case["group"]
    return v * scales.double()[:, which]


def _exact_store(s, case):
    x = s["t"]["rows"].double()
    top = LARGEST_CODE[case["format"]]
    out = torch.empty_like(x)
    scales = torch.zeros(s["t"]["scales"].shape, dtype=torch.float64, device="cuda")
    for g in range(_groups(case)):
        part = x[:, g * case["group"]:(g + 1) * case["group"]]
        scale = part.abs().max(1).values / top
        unit = part / torch.where(scale > 0, scale, 1.0)[:, None]
        if case["format"] == "fp8":
            # three bits after the leading one, 2^-9 at the least
            step = torch.exp2(torch.floor(torch.log2(unit.abs().clamp(min=2.0**-6))) - 3)
            unit = torch.round(unit / step) * step
        else:
            unit = torch.round(unit)
        out[:, g * case["group"]:(g + 1) * case["group"]] = unit * scale[:, None]
        scales[s["t"]["slots"], g] = scale
    return {"rows": out, "scales": scales}


def _exact_maxsim(s, case):
    t, page = s["t"], s["page"]
    lens, start, pages = (t[name].cpu().numpy() for name in ("doc_lens", "page_start", "pages"))
    cands, q_lens = t["cands"].cpu().numpy(), t["query_lens"].cpu().numpy()
    out = torch.full(cands.shape, float("-inf"), dtype=torch.float64, device="cuda")
    for q in range(case["nq"]):
        rows = np.flatnonzero(cands[q] >= 0)
        rows = rows[lens[cands[q][rows]] > 0]
        if not rows.size:
            continue
        docs = cands[q][rows]
        count = lens[docs].astype(np.int64)
        of = np.repeat(np.arange(rows.size), count)
        at = np.arange(int(count.sum())) - np.repeat(np.cumsum(count) - count, count)
        slot = torch.from_numpy(pages[start[docs][of] + at // page].astype(np.int64) * page + at % page).cuda()
        vectors = _exact_values(t["codes"][slot], t["scales"][slot], case)
        products = vectors @ t["queries"][q, :q_lens[q]].double().T.contiguous()
        best = torch.full((rows.size, products.shape[1]), float("-inf"), dtype=torch.float64, device="cuda")
        best.scatter_reduce_(0, torch.from_numpy(of).cuda()[:, None].expand_as(products), products, "amax")
        out[q, torch.from_numpy(rows).cuda()] = best.sum(1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("dense", "train"):
        return _exact_dense(s, case)
    if case["kind"] == "store":
        return _exact_store(s, case)
    if case["kind"] == "read":
        return _exact_values(s["t"]["codes"][s["t"]["slots"]], s["t"]["scales"][s["t"]["slots"]], case)
    return _exact_maxsim(s, case)
