"""Cases of the 8-bit floating point operators: rows quantised by blocks of 128, products with such weights, whole gated
feed-forwards, and whole layers of routed experts.  Sizes are those of the benchmark's shapes and of the tests, and ragged ones.

Format: a row's blocks of 128 values share a power of two 2^(s - 127), the smallest (s in 1 .. 247) with which the block's largest
finite magnitude is at most 448; the values are stored as e4m3, rounded to nearest even; rows are padded with zeros to whole blocks."""
import math

import torch

own = False

BLOCK = 128


def listed():
    return [
        # one token's activations before a projection: latency
        {"name": "rows_1", "op": "rows", "M": 1, "K": 5120, "type": "bfloat16", "gated": False},
        # a whole prompt portion's activations: a pass over memory
        {"name": "rows_8192", "op": "rows", "M": 8192, "K": 5120, "type": "bfloat16", "gated": False},
        # gate and up columns of an odd width in 32 bits, with the activation
        {"name": "rows_gated_odd", "op": "rows", "M": 777, "K": 1403, "type": "float32", "gated": True},
        # the fused q, k, v projection of one decoded token
        {"name": "linear_1", "op": "linear", "M": 1, "N": 7168, "K": 5120, "type": "bfloat16"},
        # the output head for a batch of thirteen requests
        {"name": "linear_head_13", "op": "linear", "M": 13, "N": 202048, "K": 5120, "type": "bfloat16"},
        # a mid-sized batch against a matrix of odd sizes, 32-bit rows
        {"name": "linear_odd_48", "op": "linear", "M": 48, "N": 4999, "K": 1900, "type": "float32"},
        # a large prompt portion against a wide matrix
        {"name": "linear_8192", "op": "linear", "M": 8192, "N": 16384, "K": 5120, "type": "bfloat16"},
        # a dense feed-forward for eight decoded tokens
        {"name": "feed_forward_8", "op": "feed_forward", "M": 8, "K": 5120, "I": 16384, "act": "silu", "type": "bfloat16"},
        # a dense feed-forward for a ragged prompt portion, a small model's sizes
        {"name": "feed_forward_3001", "op": "feed_forward", "M": 3001, "K": 2048, "I": 2816, "act": "gelu_tanh", "type": "bfloat16"},
        # one decoded token through one of sixteen experts and the shared one, its score on the experts' input
        {"name": "experts_1", "op": "experts", "M": 1, "K": 5120, "I": 8192, "E": 16, "k": 1, "on_input": True, "shared": True,
         "act": "silu", "type": "bfloat16"},
        # eight decoded tokens, six picks each of sixty-four narrow experts, weights where the outputs are summed
        {"name": "experts_8_of_64", "op": "experts", "M": 8, "K": 2048, "I": 1408, "E": 64, "k": 6, "on_input": False, "shared": False,
         "act": "silu", "type": "bfloat16"},
        # a prompt portion through sixteen wide experts and the shared one
        {"name": "experts_2048", "op": "experts", "M": 2048, "K": 5120, "I": 8192, "E": 16, "k": 1, "on_input": True, "shared": True,
         "act": "silu", "type": "bfloat16"},
    ]


def draw(rng):
    def size(lo, hi, odd):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return v if odd else max(128, v // 128 * 128)
    op = rng.choice(["rows", "linear", "linear", "feed_forward", "experts", "experts"])
    odd = rng.random() < 0.4
    c = {"op": op, "type": rng.choice(["bfloat16", "bfloat16", "float32"]), "M": size(1, 8192, True)}
    if op == "rows":
        c.update(K=size(130, 8192, odd), gated=rng.random() < 0.4)
    elif op == "linear":
        c.update(K=size(200, 14000, odd), N=size(200, 28000, odd))
        c["M"] = max(1, min(c["M"], int(2e11 / (c["K"] * c["N"]))))
    elif op == "feed_forward":
        c.update(K=size(300, 5120, odd), I=size(300, 16384, odd), act=rng.choice(["silu", "gelu_tanh"]))
        c["M"] = max(1, min(c["M"], int(1e11 / (c["K"] * c["I"]))))
    else:
        E = rng.choice([4, 8, 16, 28, 32, 64, 100])
        c.update(E=E, k=rng.choice([1, 2, 4, 6] if E >= 8 else [1, 2]), on_input=rng.random() < 0.4, shared=rng.random() < 0.4,
                 act=rng.choice(["silu", "gelu_tanh"]), K=size(300, 5120, odd), I=size(300, 5120, odd), M=size(1, 2500, True))
        while (E + 1) * c["K"] * c["I"] > 6e8:
            c["K"], c["I"] = c["K"] // 2, c["I"] // 2
        c["M"] = max(1, min(c["M"], int(6e10 / (c["K"] * c["I"] * (c["k"] + 1)))))
    return c


def _blocks(K):
    return -(-K // BLOCK)


def _inputs(case, seed):
    """Activations as they come from a norm (a few channels larger than the rest), stored codes and scale bytes of weights around
    0.02, and a router's picks with their weights."""
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)
    op, M, K = case["op"], case["M"], case["K"]
    kind = getattr(torch, case["type"])

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def matrix(*shape):
        codes = torch.empty(*shape, dtype=torch.float8_e4m3fn, device="cuda")
        for part in (codes if len(shape) > 2 else [codes]):
            part.copy_((normal(*part.shape) * 130.0).clamp_(-448.0, 448.0))
        return codes, torch.randint(113, 116, (*shape[:-1], _blocks(shape[-1])), generator=g, device="cuda", dtype=torch.uint8)
    s = {}
    cols = 2 * K if case.get("gated") else K
    s["x"] = (normal(M, cols) * torch.exp(0.7 * normal(cols))).to(kind)
    if op == "linear":
        s["w"] = matrix(case["N"], K)
    elif op == "feed_forward":
        s["w1"], s["w2"] = matrix(2 * case["I"], K), matrix(K, case["I"])
    elif op == "experts":
        n = case["E"] + (1 if case["shared"] else 0)
        s["w1"], s["w2"] = matrix(n, 2 * case["I"], K), matrix(n, K, case["I"])
        logits = normal(M, case["E"]) + 0.5 * normal(case["E"])
        top, ids = torch.topk(logits, case["k"], dim=1)
        s["ids"] = ids.to(torch.int32).contiguous()
        s["wts"] = (torch.sigmoid(top) if case["on_input"] else torch.softmax(top, dim=1)).contiguous()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from sharpinference_amd import ops
        if "w" in s:
            s["w"] = ops.fp8_weight(*s["w"])
        if "w1" in s:
            s["w1"], s["w2"] = ops.fp8_weight(*s["w1"], gated=True), ops.fp8_weight(*s["w2"])
        s["code"] = {"silu": ops.ACT_SILU, "gelu_tanh": ops.ACT_GELU_TANH}.get(case.get("act", "silu"))
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------------
def _act(name, g, u):
    if name == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g))) * u
    return g / (1.0 + torch.exp(-g)) * u


def _quantised(x):
    """(codes e4m3 [M, whole blocks], scale bytes [M, blocks]) of the rows of x."""
    M, K = x.shape
    B = _blocks(K)
    v = torch.nn.functional.pad(x.float(), (0, B * BLOCK - K)).view(M, B, BLOCK)
    finite = torch.isfinite(v)
    bits = torch.where(finite, v.abs(), torch.zeros_like(v)).amax(2).view(torch.int32)
    s = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(1, 247)
    inverse = ((254 - s) << 23).view(torch.float32)
    v = torch.where(finite, v * inverse[..., None], torch.full_like(v, float("nan")))
    return v.to(torch.float8_e4m3fn).view(M, B * BLOCK), s.to(torch.uint8)


def _values(codes, scales):
    """float32 values of stored codes [.., K] and bytes [.., blocks]."""
    K = codes.shape[-1]
    p = (scales.int() << 23).view(torch.float32)
    return codes.float() * p.repeat_interleave(BLOCK, dim=-1)[..., :K]


def _rounded_rows(x):
    return _values(*_quantised(x))[:, :x.shape[1]]


def _feed_forward(xq, w1, w2, act, score=None):
    y = xq @ _values(*w1).t()
    if score is not None:
        y = y * score[:, None]
    g, u = y.chunk(2, dim=1)
    h = _act(act, g, u).to(torch.bfloat16)
    return _rounded_rows(h) @ _values(*w2).t()


def run(state):
    c = state["case"]
    if own:
        from sharpinference_amd import ops
        if c["op"] == "rows":
            q = ops.quantize_rows(state["x"], act=state["code"] if c["gated"] else None)
            return {"codes": q.codes, "scales": q.scales[:, :_blocks(c["K"])]}
        if c["op"] == "linear":
            return ops.linear_fp8(state["x"], state["w"])
        if c["op"] == "feed_forward":
            return ops.feed_forward_fp8(state["x"], state["w1"], state["w2"], act=state["code"])
        return ops.experts_fp8(state["x"], state["ids"], state["wts"], state["w1"], state["w2"], act=state["code"],
                               score_on_input=c["on_input"], shared=c["shared"])
    x = state["x"]
    if c["op"] == "rows":
        if c["gated"]:
            g, u = x.float().chunk(2, dim=1)
            x = _act("silu", g, u).to(x.dtype)
        codes, scales = _quantised(x)
        return {"codes": codes, "scales": scales}
    xq = _rounded_rows(x)
    if c["op"] == "linear":
        return (xq @ _values(*state["w"]).t()).to(torch.bfloat16)
    if c["op"] == "feed_forward":
        return _feed_forward(xq, state["w1"], state["w2"], c["act"]).to(torch.bfloat16)
    w1, w2, ids, wts = state["w1"], state["w2"], state["ids"], state["wts"]
    out = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    for e in range(c["E"]):
        rows, place = torch.nonzero(ids == e, as_tuple=True)
        if rows.numel() == 0:
            continue
        weight = wts[rows, place]
        y = _feed_forward(xq[rows], (w1[0][e], w1[1][e]), (w2[0][e], w2[1][e]), c["act"], weight if c["on_input"] else None)
        out.index_add_(0, rows, y if c["on_input"] else y * weight[:, None])
    if c["shared"]:
        e = c["E"]
        out += _feed_forward(xq, (w1[0][e], w1[1][e]), (w2[0][e], w2[1][e]), c["act"])
    return out.to(torch.bfloat16)


def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    size = 2 if case["type"] == "bfloat16" else 4
    if op == "rows":
        cols = 2 * K if case["gated"] else K
        return {"bytes": M * (cols * size + _blocks(K) * (BLOCK + 1)), "flops": M * cols * 2}

    def matrix(rows, cols):
        return rows * (cols + _blocks(cols))
    if op == "linear":
        N = case["N"]
        return {"bytes": matrix(N, K) + M * (K * size + 2 * N), "flops": 2 * M * N * K}
    per = matrix(2 * case["I"], K) + matrix(K, case["I"])
    if op == "feed_forward":
        return {"bytes": per + M * K * (size + 2), "flops": 6 * M * K * case["I"]}
    E, k = case["E"], case["k"]
    met = E * (1.0 - (1.0 - k / E) ** M) + (1 if case["shared"] else 0)        # experts that some token picks, on average
    return {"bytes": int(met * per) + M * (K * (size + 2) + 8 * k), "flops": 6 * M * (k + (1 if case["shared"] else 0)) * K * case["I"]}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def _power(e):
    """2^e in 64 bits, exactly (e from -1022 on)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_blocks(v):
    """Codes (as numbers) and exponents of rows given in 64 bits, padded to whole blocks."""
    M, K = v.shape
    B = _blocks(K)
    whole = torch.zeros(M, B * BLOCK, dtype=torch.float64, device=v.device)
    whole[:, :K] = v
    whole = whole.reshape(M, B, BLOCK)
    top = whole.abs().max(dim=2).values
    mantissa, power = torch.frexp(top)                       # top = mantissa 2^power, 448 = 0.875 2^9
    e = torch.where(mantissa <= 0.875, power - 9, power - 8)
    e = torch.where(top > 0, e, torch.full_like(e, -126)).clamp(-126, 120)
    scaled = whole * _power(-e)[..., None]
    _, p = torch.frexp(scaled)
    step = _power(torch.clamp(p - 1, min=-6) - 3)       # four bits of a value, steps of 2^-9 at least
    return torch.round(scaled / step) * step, e


def _exact_rows(v):
    codes, e = _exact_blocks(v)
    return (codes * _power(e)[..., None]).reshape(v.shape[0], -1)[:, :v.shape[1]]


def _exact_weight(w):
    codes, scales = w
    e = (scales.to(torch.int32) - 127).unsqueeze(-1).expand(*scales.shape, BLOCK).reshape(scales.shape[0], -1)[:, :codes.shape[1]]
    return codes.to(torch.float64) * _power(e)


def _exact_unit(name, g, u):
    if name == "gelu_tanh":
        return u * g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
    return u * g * torch.sigmoid(g)


def exact(case, seed):
    s = _inputs(case, seed)
    x, op = s["x"].double(), case["op"]
    if op == "rows":
        if case["gated"]:
            half = x.shape[1] // 2
            x = _exact_unit("silu", x[:, :half], x[:, half:])
            if case["type"] == "bfloat16":
                x = x.to(torch.bfloat16).double()
        codes, e = _exact_blocks(x)
        return {"codes": codes.reshape(x.shape[0], -1), "scales": (e + 127).to(torch.uint8)}
    xe = _exact_rows(x)
    if op == "linear":
        return torch.matmul(xe, _exact_weight(s["w"]).T)

    def unit(rows, a, b, score):
        both = torch.matmul(rows, _exact_weight(a).T) * score
        half = both.shape[1] // 2
        h = _exact_unit(case["act"], both[:, :half], both[:, half:]).to(torch.bfloat16).double()
        return torch.matmul(_exact_rows(h), _exact_weight(b).T)
    if op == "feed_forward":
        return unit(xe, s["w1"], s["w2"], 1.0)
    total = torch.zeros_like(x)
    for e in range(case["E"] + (1 if case["shared"] else 0)):
        a, b = (s["w1"][0][e], s["w1"][1][e]), (s["w2"][0][e], s["w2"][1][e])
        if e == case["E"]:
            total += unit(xe, a, b, 1.0)
            continue
        for j in range(case["k"]):
            at = torch.nonzero(s["ids"][:, j] == e).flatten()
            if at.numel():
                weight = s["wts"][at, j].double().unsqueeze(1)
                y = unit(xe[at], a, b, weight if case["on_input"] else 1.0)
                total[at] += y if case["on_input"] else y * weight
    return total
