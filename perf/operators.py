"""Measured calls of the training and answering operators around a language model's matrix products: layer norm, embedding,
log probabilities of tokens, and clipping by the global norm; each in its plain form (elementary torch operations) and as
the calls a user makes of the library's entry points."""
import ctypes

import torch

own = False

TYPES = {"Float": torch.float32, "Half": torch.float16, "Double": torch.float64}
BYTES = {"Float": 4, "Half": 2, "Double": 8}


def _compute(t):
    return torch.float64 if t == torch.float64 else torch.float32


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoding step of a few sequences: latency is all there is
        {"name": "layernorm_4x768_float", "op": "layernorm", "type": "Float", "rows": 4, "length": 768, "pad": 0, "affine": True},
        # a training batch's activations, storage in half
        {"name": "layernorm_16384x1024_half", "op": "layernorm", "type": "Half", "rows": 16384, "length": 1024, "pad": 0, "affine": True},
        # the backward pass of such a batch, in float
        {"name": "layernorm_bp_16384x1024_float", "op": "layernorm_bp", "type": "Float", "rows": 16384, "length": 1024, "pad": 0, "affine": True},
        # an odd batch of odd rows: no row but the first starts on a vector's boundary
        {"name": "layernorm_bp_4097x5003_half", "op": "layernorm_bp", "type": "Half", "rows": 4097, "length": 5003, "pad": 0, "affine": True},
        # the tokens of a batch looked up
        {"name": "embedding_32768x1024_half", "op": "embedding", "type": "Half", "n": 32768, "vocabulary": 50257, "length": 1024, "padding": 0.02},
        # the table's gradient for a batch: frequent tokens come thousands of times, most never
        {"name": "embedding_bp_16384x768_float", "op": "embedding_bp", "type": "Float", "n": 16384, "vocabulary": 32000, "length": 768, "padding": 0.02},
        # a small table of a gradient check, in double, odd everywhere
        {"name": "embedding_bp_257x65_double", "op": "embedding_bp", "type": "Double", "n": 257, "vocabulary": 1000, "length": 65, "padding": 0.02},
        # answering: the next token's distribution of one sequence, with alternatives; the vocabulary's padding is masked
        {"name": "logprobs_1x50257_half_top8", "op": "logprobs", "type": "Half", "rows": 1, "length": 50257, "pad": 0, "k": 8, "masked": 17},
        # scoring a batch of answers
        {"name": "logprobs_4096x32000_float_top5", "op": "logprobs", "type": "Float", "rows": 4096, "length": 32000, "pad": 0, "k": 5, "masked": 0},
        # the loss's gradient on a batch, rows of an odd vocabulary
        {"name": "logprobs_bp_4096x50257_half", "op": "logprobs_bp", "type": "Half", "rows": 4096, "length": 50257, "pad": 0, "entropy": False},
        # a small model's gradients, views into one vector
        {"name": "clip_20_small_half", "op": "clip", "type": "Half", "count": 20, "total": 100003, "flat": True},
        # the gradients of a model of ordinary size, tensors of their own
        {"name": "clip_60_large_float", "op": "clip", "type": "Float", "count": 60, "total": 124000000, "flat": False},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["layernorm", "layernorm_bp", "embedding", "embedding_bp", "logprobs", "logprobs_bp", "clip"])
    kind = rng.choice(["Float", "Half", "Double"])
    most = 400000000 // BYTES[kind]  # elements of the largest operand
    case = {"op": op, "type": kind}
    if op.startswith("layernorm"):
        case["length"] = _spread(rng, 8, 16384)
        case["rows"] = _spread(rng, 1, max(1, min(16384, most // 12 // case["length"])))
        case["pad"] = rng.choice([0, 0, 8, 3])
        case["affine"] = rng.random() < 0.8
    elif op.startswith("embedding"):
        case["length"] = _spread(rng, 1, 2048)
        case["n"] = _spread(rng, 1, max(1, min(65536, most // 6 // case["length"])))
        case["vocabulary"] = _spread(rng, 16, max(16, min(100000, most // 4 // case["length"])))
        case["padding"] = rng.choice([0.0, 0.02, 0.5])
    elif op.startswith("logprobs"):
        case["length"] = _spread(rng, 16, 131072)
        case["rows"] = _spread(rng, 1, max(1, min(8192, most // 4 // case["length"])))
        case["pad"] = rng.choice([0, 0, 8, 3])
        if op == "logprobs":
            case["k"] = rng.choice([0, 1, 5, 8, 16])
            case["masked"] = rng.choice([0, 0, 5])
        else:
            case["entropy"] = rng.random() < 0.3
    else:
        case["count"] = rng.randint(1, 60)
        case["total"] = _spread(rng, 1000, most // 2)
        case["flat"] = rng.random() < 0.5
    return case


def work(case):
    b = BYTES[case["type"]]
    c = 8 if b == 8 else 4
    op = case["op"]
    if op == "layernorm":
        e = case["rows"] * case["length"]
        return {"bytes": 2 * e * b + 2 * case["rows"] * c + 2 * case["length"] * b, "flops": 8 * e}
    if op == "layernorm_bp":
        e = case["rows"] * case["length"]
        return {"bytes": 3 * e * b + 2 * case["rows"] * c + 3 * case["length"] * b, "flops": 14 * e}
    if op == "embedding":
        e = case["n"] * case["length"]
        return {"bytes": 2 * e * b + 8 * case["n"], "flops": e}
    if op == "embedding_bp":
        e = case["n"] * case["length"]
        return {"bytes": e * b + case["vocabulary"] * case["length"] * b + 8 * case["n"], "flops": 2 * e}
    if op == "logprobs":
        e = case["rows"] * case["length"]
        return {"bytes": e * b + case["rows"] * (8 + 3 * c + case["k"] * (8 + c)), "flops": 7 * e}
    if op == "logprobs_bp":
        e = case["rows"] * case["length"]
        return {"bytes": 2 * e * b + case["rows"] * (8 + 4 * c), "flops": 6 * e}
    return {"bytes": 2 * case["total"] * b, "flops": 3 * case["total"]}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _info(rows, cols, pitch):
    """A matrix's shapeInfo: rank, shape, strides, offset, element-wise stride, order."""
    return torch.tensor([2, rows, cols, pitch, 1, 0, 1 if rows == 1 or pitch == cols else -1, 99], dtype=torch.int64)


def _matrix(rows, length, pad, dtype, g, scale=1.0):
    """A random matrix whose rows lie length + pad elements apart."""
    m = torch.randn(rows, length + pad, device="cuda", generator=g, dtype=torch.float32).mul_(scale).to(dtype)
    return m[:, :length]


def _tokens(n, vocabulary, padding, g):
    """Token numbers as text has them (the r-th most frequent about 1 / r as frequent as the first), some of them padding."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    t = (float(vocabulary + 1) ** u).long().sub_(1).clamp_(0, vocabulary - 1)
    t = t * 7919 % vocabulary if vocabulary % 7919 else t
    return torch.where(torch.rand(n, device="cuda", generator=g) < padding, torch.full_like(t, -1), t)


def _lengths(count, total):
    """Ragged lengths of `count` tensors, `total` elements in all, none of them empty."""
    r = torch.rand(count, generator=torch.Generator().manual_seed(count + total), dtype=torch.float64).pow_(3).add_(1e-4)
    n = (r / r.sum() * (total - count)).long().add_(1)
    n[-1] += total - int(n.sum())
    return n.tolist()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    c = _compute(dtype)
    op = case["op"]
    s = {"case": case, "op": op, "type": case["type"]}
    if op.startswith("layernorm"):
        rows, length, pad = case["rows"], case["length"], case["pad"]
        s["x"] = _matrix(rows, length, pad, dtype, g, 2.0).add_(0.5)
        s["info"], s["dense"] = _info(rows, length, length + pad), _info(rows, length, length)
        s["gain"] = s["bias"] = None
        if case["affine"]:
            s["gain"] = torch.randn(length, device="cuda", generator=g).mul_(0.1).add_(1.0).to(dtype)
            s["bias"] = torch.randn(length, device="cuda", generator=g).mul_(0.1).to(dtype)
        s["mean"], s["inv_std"] = (torch.empty(rows, dtype=c, device="cuda") for _ in range(2))
        if op == "layernorm":
            s["z"] = torch.empty(rows, length, dtype=dtype, device="cuda")
        else:
            s["dz"] = torch.randn(rows, length, device="cuda", generator=g).mul_(0.1).to(dtype)
            x = s["x"].double()
            s["mean"].copy_(x.mean(1))
            s["inv_std"].copy_((x.var(1, unbiased=False) + 1e-5).rsqrt())
            s["dx"] = torch.empty(rows, length, dtype=dtype, device="cuda")
            s["dgain"], s["dbias"] = (torch.empty(length, dtype=dtype, device="cuda") for _ in range(2))
    elif op.startswith("embedding"):
        n, v, length = case["n"], case["vocabulary"], case["length"]
        s["tokens"] = _tokens(n, v, case["padding"], g)
        s["scale"] = float(length) ** 0.5
        s["rows_info"], s["table_info"] = _info(n, length, length), _info(v, length, length)
        if op == "embedding":
            s["table"] = _matrix(v, length, 0, dtype, g, 0.02)
            s["z"] = torch.empty(n, length, dtype=dtype, device="cuda")
        else:
            s["dz"] = _matrix(n, length, 0, dtype, g, 0.1)
            s["dtable"] = torch.empty(v, length, dtype=dtype, device="cuda")
    elif op.startswith("logprobs"):
        rows, length, pad = case["rows"], case["length"], case["pad"]
        s["x"] = _matrix(rows, length, pad, dtype, g, 2.5)
        s["info"], s["dense"] = _info(rows, length, length + pad), _info(rows, length, length)
        s["tokens"] = torch.randint(0, length - case.get("masked", 0), (rows,), device="cuda", generator=g)
        if op == "logprobs":
            if case["masked"]:
                s["x"][:, length - case["masked"]:] = float("-inf")
            s["k"] = case["k"]
            s["lp"], s["log_sum"], s["entropy"] = (torch.empty(rows, dtype=c, device="cuda") for _ in range(3))
            s["top"] = torch.empty(rows, case["k"], dtype=torch.int64, device="cuda")
            s["top_lp"] = torch.empty(rows, case["k"], dtype=c, device="cuda")
        else:
            s["tokens"][torch.rand(rows, device="cuda", generator=g) < 0.05] = -1  # padded positions
            s["d_lp"] = torch.randn(rows, device="cuda", generator=g).to(c)
            s["d_entropy"] = torch.randn(rows, device="cuda", generator=g).mul_(0.01).to(c) if case["entropy"] else None
            s["log_sum"] = torch.logsumexp(s["x"].to(c), 1)
            lp = s["x"].to(c) - s["log_sum"][:, None]
            s["entropy"] = -(lp.exp() * lp).sum(1)
            del lp
            s["dx"] = torch.empty(rows, length, dtype=dtype, device="cuda")
    else:
        lengths = _lengths(case["count"], case["total"])
        flat = torch.randn(case["total"], device="cuda", generator=g, dtype=torch.float32).mul_(0.01).to(dtype)
        out = torch.empty_like(flat)
        s["g"], s["z"] = list(flat.split(lengths)), list(out.split(lengths))
        if not case["flat"]:
            s["g"], s["z"] = [t.clone() for t in s["g"]], [torch.empty_like(t) for t in s["z"]]
        s["tables"] = torch.tensor([[t.data_ptr() for t in s["g"]], [t.data_ptr() for t in s["z"]]], dtype=torch.int64, device="cuda")
        ends = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0)
        s["offsets"], s["total"] = ends.cuda(), case["total"]
        s["norm"] = torch.empty(1, dtype=c, device="cuda")
        s["max_norm"] = 1.0
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _plain_layernorm(s):
    c = _compute(s["x"].dtype)
    x = s["x"].to(c)
    mean = x.mean(1, keepdim=True)
    d = x - mean
    inv = 1.0 / ((d * d).mean(1, keepdim=True) + 1e-5).sqrt()
    z = d * inv
    if s["gain"] is not None:
        z = z * s["gain"].to(c) + s["bias"].to(c)
    return z.to(s["x"].dtype), mean[:, 0], inv[:, 0]


def _plain_layernorm_bp(s):
    t = s["x"].dtype
    c = _compute(t)
    dz = s["dz"].to(c)
    inv = s["inv_std"][:, None]
    h = (s["x"].to(c) - s["mean"][:, None]) * inv
    a = dz if s["gain"] is None else dz * s["gain"].to(c)
    dx = inv * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    return dx.to(t), (dz * h).sum(0).to(t), dz.sum(0).to(t)


def _plain_embedding(s):
    c = _compute(s["table"].dtype)
    t = s["tokens"]
    rows = s["table"][t.clamp(min=0)].to(c) * s["scale"]
    return torch.where((t < 0)[:, None], torch.zeros((), dtype=c, device=rows.device), rows).to(s["table"].dtype)


def _plain_embedding_bp(s):
    c = _compute(s["dz"].dtype)
    v = s["case"]["vocabulary"]
    t = s["tokens"]
    into = torch.where(t < 0, torch.full_like(t, v), t)  # padding goes to a row behind the table
    d = torch.zeros(v + 1, s["dz"].shape[1], dtype=c, device=t.device)
    d.index_add_(0, into, s["dz"].to(c))
    return (d[:v] * s["scale"]).to(s["dz"].dtype)


def _top(x, k):
    """The k largest of every row, the lowest index first among equals."""
    if x.dtype == torch.float64:
        return torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    bits = (x.float() + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32)  # whole numbers in the order of the values
    key += (1 << 32) - 1 - torch.arange(x.shape[1], device=x.device)
    return (1 << 32) - 1 - (torch.topk(key, k, dim=1)[0] & 0xFFFFFFFF)


def _plain_logprobs(s):
    c = _compute(s["x"].dtype)
    x = s["x"].to(c)
    m = x.amax(1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(1)
    log_sum = m[:, 0] + total.log()
    entropy = total.log() - torch.where(e > 0, d * e, torch.zeros_like(e)).sum(1) / total
    lp = x.gather(1, s["tokens"][:, None])[:, 0] - log_sum
    if not s["k"]:
        return lp, log_sum, entropy
    top = _top(s["x"], s["k"])
    return lp, log_sum, entropy, top, x.gather(1, top) - log_sum[:, None]


def _plain_logprobs_bp(s):
    c = _compute(s["x"].dtype)
    t = s["tokens"]
    d = torch.where(t < 0, torch.zeros_like(s["d_lp"]), s["d_lp"])[:, None]
    lp = s["x"].to(c) - s["log_sum"][:, None]
    p = lp.exp()
    dx = -d * p
    if s["d_entropy"] is not None:
        dx = dx - s["d_entropy"][:, None] * p * (lp + s["entropy"][:, None])
    dx.scatter_add_(1, t.clamp(min=0)[:, None], d)
    return dx.to(s["x"].dtype)


def _plain_clip(s):
    c = _compute(s["g"][0].dtype)
    norm = torch.stack([t.to(c).square().sum(dtype=torch.float64) for t in s["g"]]).sum().sqrt()
    factor = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).to(c)
    return [(t.to(c) * factor).to(t.dtype) for t in s["g"]], norm.to(c).reshape(1)


# ---- the library's calls ---------------------------------------------------------------------------------------------

_native = None


def _ops():
    global _native
    if _native is None:
        from libnd4j_amd.native import NativeOps
        _native = NativeOps()
    return _native


def _extra(x=None, y=None, z=None):
    e = (ctypes.c_void_p * 20)()
    e[1] = torch.cuda.current_stream().cuda_stream
    if x is not None:
        e[0] = x.data_ptr()
    if y is not None:
        e[7] = y.data_ptr()
    if z is not None:
        e[8] = z.data_ptr()
    return e


def _at(t):
    return None if t is None else t.data_ptr()


def _own_layernorm(s):
    call = getattr(_ops(), "amd_execLayerNorm" + s["type"])
    call(_extra(x=s["info"], z=s["dense"]), _at(s["x"]), _at(s["info"]), _at(s["gain"]), _at(s["bias"]), _at(s["z"]), _at(s["dense"]),
         _at(s["mean"]), _at(s["inv_std"]), 1e-5)
    return s["z"], s["mean"], s["inv_std"]


def _own_layernorm_bp(s):
    call = getattr(_ops(), "amd_execLayerNormBp" + s["type"])
    call(_extra(x=s["info"], y=s["dense"], z=s["dense"]), _at(s["x"]), _at(s["info"]), _at(s["gain"]), _at(s["mean"]), _at(s["inv_std"]),
         _at(s["dz"]), _at(s["dense"]), _at(s["dx"]), _at(s["dense"]), _at(s["dgain"]), _at(s["dbias"]), None, 0)
    return s["dx"], s["dgain"], s["dbias"]


def _own_embedding(s):
    call = getattr(_ops(), "amd_execEmbedding" + s["type"])
    call(_extra(x=s["table_info"], z=s["rows_info"]), _at(s["table"]), _at(s["table_info"]), _at(s["tokens"]), s["case"]["n"], _at(s["z"]),
         _at(s["rows_info"]), s["scale"])
    return s["z"]


def _own_embedding_bp(s):
    call = getattr(_ops(), "amd_execEmbeddingBp" + s["type"])
    call(_extra(x=s["rows_info"], z=s["table_info"]), _at(s["dz"]), _at(s["rows_info"]), _at(s["tokens"]), s["case"]["n"], _at(s["dtable"]),
         _at(s["table_info"]), s["scale"], 0, None, 0)
    return s["dtable"]


def _own_logprobs(s):
    call = getattr(_ops(), "amd_execTokenLogProbs" + s["type"])
    call(_extra(x=s["info"]), _at(s["x"]), _at(s["info"]), _at(s["tokens"]), _at(s["lp"]), _at(s["log_sum"]), _at(s["entropy"]), s["k"],
         _at(s["top"]), _at(s["top_lp"]), None, 0)
    return (s["lp"], s["log_sum"], s["entropy"], s["top"], s["top_lp"]) if s["k"] else (s["lp"], s["log_sum"], s["entropy"])


def _own_logprobs_bp(s):
    call = getattr(_ops(), "amd_execTokenLogProbsBp" + s["type"])
    call(_extra(x=s["info"], z=s["dense"]), _at(s["x"]), _at(s["info"]), _at(s["tokens"]), _at(s["log_sum"]), _at(s["entropy"]), _at(s["d_lp"]),
         _at(s["d_entropy"]), _at(s["dx"]), _at(s["dense"]))
    return s["dx"]


def _own_clip(s):
    call = getattr(_ops(), "amd_execClipByGlobalNorm" + s["type"])
    tables = s["tables"].data_ptr()
    count = s["case"]["count"]
    call(_extra(), tables, tables + 8 * count, _at(s["offsets"]), count, s["total"], s["max_norm"], _at(s["norm"]), None, 0)
    return s["z"], s["norm"]


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["op"]](state)


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("layernorm"):
        x = s["x"].double()
        gain = torch.ones(x.shape[1], dtype=torch.float64, device="cuda") if s["gain"] is None else s["gain"].double()
        if op == "layernorm":
            mean = x.sum(1) / x.shape[1]
            std = ((x - mean[:, None]).pow(2).sum(1) / x.shape[1] + 1e-5).sqrt()
            z = (x - mean[:, None]) / std[:, None] * gain
            return z if s["bias"] is None else z + s["bias"].double(), mean, 1 / std
        dz, inv = s["dz"].double(), s["inv_std"].double()[:, None]
        h = (x - s["mean"].double()[:, None]) * inv
        a = dz * gain
        n = x.shape[1]
        dx = (n * a - a.sum(1, keepdim=True) - h * (a * h).sum(1, keepdim=True)) * inv / n
        return dx, torch.linalg.vecdot(dz, h, dim=0), dz.sum(0)
    if op == "embedding":
        t = s["tokens"]
        z = s["table"].double().index_select(0, t.clamp(min=0)).mul_(s["scale"])
        z[t < 0] = 0
        return z
    if op == "embedding_bp":
        order = torch.argsort(s["tokens"], stable=True)
        t = s["tokens"][order]
        sums = torch.cat([torch.zeros(1, case["length"], dtype=torch.float64, device="cuda"), s["dz"].double()[order].cumsum(0)])
        ids = torch.arange(case["vocabulary"], device="cuda")
        return (sums[torch.searchsorted(t, ids, right=True)] - sums[torch.searchsorted(t, ids)]) * s["scale"]
    if op == "logprobs":
        logp = torch.log_softmax(s["x"].double(), 1)
        log_sum = torch.logsumexp(s["x"].double(), 1)
        entropy = torch.special.entr(logp.exp()).sum(1)
        lp = logp[torch.arange(case["rows"], device="cuda"), s["tokens"]]
        if not case["k"]:
            return lp, log_sum, entropy
        value, top = torch.sort(s["x"], dim=1, descending=True, stable=True)
        return lp, log_sum, entropy, top[:, :case["k"]].contiguous(), value[:, :case["k"]].double() - log_sum[:, None]
    if op == "logprobs_bp":
        x = s["x"].double()
        logp = x - s["log_sum"].double()[:, None]
        one = torch.zeros_like(x)
        live = s["tokens"] >= 0
        one[live, s["tokens"][live]] = 1.0
        p = logp.exp_()
        dx = (one - live[:, None] * p).mul_(s["d_lp"].double()[:, None])
        if s["d_entropy"] is not None:
            dx += s["d_entropy"].double()[:, None] * (torch.special.entr(p) - p * s["entropy"].double()[:, None])
        return dx
    flat = torch.cat([t.double() for t in s["g"]])
    norm = torch.linalg.vector_norm(flat)
    factor = min(1.0, s["max_norm"] / float(norm))
    return [t.double() * factor for t in s["g"]], norm.reshape(1)
