"""The low-precision and mixture-of-experts operators, one call each, in plain torch form and through the
runtime's entry points.

A case is one pass through one operator:

quantise   rows of fp32 / bf16 / fp16 to e4m3 with a power-of-two scale for each block of 128 along the row
           (activations; rows may be gathered by an index on the way) or of 128 x 128 (weights)
product    out = act(A B^T + bias) of e4m3 operands with an fp32 scale for each block: 1 x 128 of A, 128 x 128 of B
grouped    the same for rows that come in ragged groups, each with a matrix of its own, in bf16, fp16 or block-scaled
           e4m3; "gated" takes two matrices for each group and gives silu(gate) * up
route      logits -> the k chosen experts of each token, their softmax weights and the order of rows by expert
combine    each token's weighted sum of its experts' rows
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
CODES = {"fp32": 0, "bf16": 1, "fp16": 2, "e4m3": 3}
ACTS = {"sigmoid": 0, "relu": 1, "tanh": 2, "none": 5, "silu": 6, "gated": 7}
BLOCK = 128
E4M3_MAX = 448.0


def _quantise(name, rows, cols, type, block_rows=1, sources=0):
    """`sources`: rows of the input when the output's rows are gathered from it, else 0."""
    return {"name": name, "op": "quantise", "rows": rows, "cols": cols, "type": type, "block_rows": block_rows,
            "sources": sources}


def _product(name, rows, n, k, out, act="none", bias=False):
    return {"name": name, "op": "product", "rows": rows, "n": n, "k": k, "out": out, "act": act, "bias": bias}


def _grouped(name, rows, groups, n, k, type, out, act="none", bias=False, sources=0):
    return {"name": name, "op": "grouped", "rows": rows, "groups": groups, "n": n, "k": k, "type": type, "out": out,
            "act": act, "bias": bias, "sources": sources}


def _route(name, tokens, experts, k, type, normalise, padded=0):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "k": k, "type": type,
            "normalise": normalise, "padded": padded}


def _combine(name, tokens, k, n, type, out):
    return {"name": name, "op": "combine", "tokens": tokens, "k": k, "n": n, "type": type, "out": out}


def listed():
    return [
        # a prompt's tokens on their way into an expert layer: each goes to four experts
        _quantise("quantise_gathered_tokens", 16384, 4096, "bf16", sources=4096),
        # VGG-16's first classifier layer, when its weights are laid out
        _quantise("quantise_fc_weights", 4096, 25088, "fp32", block_rows=128),
        # the same layer with 8-bit weights: one image, a batch of 64
        _product("product_fc_one_image", 1, 4096, 25088, "fp32", "relu", True),
        _product("product_fc_batch64", 64, 4096, 25088, "bf16", "relu", True),
        # a dense layer over a long prompt
        _product("product_prompt", 8190, 8192, 4096, "bf16"),
        # expert layer, first product: 32 sequences that take one token each, four experts a token
        _grouped("grouped_tokens_bf16", 128, 64, 1024, 2048, "bf16", "bf16", "gated", sources=32),
        # the same layer over a prompt, in 8 bits
        _grouped("grouped_prompt_e4m3", 16384, 32, 1024, 2048, "e4m3", "bf16", "gated", sources=4096),
        # a few groups of odd sizes, fp32 results
        _grouped("grouped_odd_fp16", 5003, 8, 1000, 1160, "fp16", "fp32", "relu", True),
        # routers: one token of each sequence; a prompt of a padded batch
        _route("route_tokens", 32, 64, 4, "fp32", True),
        _route("route_prompt", 16384, 128, 8, "bf16", True, padded=37),
        # the experts' rows back at their tokens
        _combine("combine_tokens", 32, 4, 2048, "bf16", "bf16"),
        _combine("combine_prompt", 16384, 4, 2048, "bf16", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "grouped", "grouped", "route", "combine"])
    if op == "quantise":
        block_rows = rng.choice([1, 1, 128])
        cols = _log_int(rng, 100, 25088)
        rows = _log_int(rng, 1, min(16384, 10 ** 8 // cols))
        sources = _log_int(rng, 1, rows) if block_rows == 1 and rng.random() < 0.5 else 0
        return _quantise("", rows, cols, rng.choice(["bf16", "fp16", "fp32"]), block_rows, sources)
    if op == "product":
        n, k = _log_int(rng, 64, 8192), _log_int(rng, 128, 25088)
        rows = _log_int(rng, 1, max(1, min(8190, int(2.7e11 / (n * k)))))
        return _product("", rows, n, k, rng.choice(["bf16", "fp16", "fp32"]),
                        rng.choice(["none", "relu", "silu", "tanh", "sigmoid"]), rng.random() < 0.5)
    if op == "grouped":
        type = rng.choice(["bf16", "fp16", "e4m3", "e4m3"])
        act = rng.choice(["none", "relu", "silu", "gated", "gated"])
        groups = _log_int(rng, 1, 64)
        n, k = 8 * _log_int(rng, 8, 256), 8 * _log_int(rng, 16, 512)
        both = 2 if act == "gated" else 1
        while groups * n * k * both > 3e8:
            groups = groups // 2 + groups % 2
        rows = _log_int(rng, 1, max(1, min(16384, int(6.8e10 / (n * k * both)))))
        sources = _log_int(rng, 1, rows) if rng.random() < 0.5 else 0
        return _grouped("", rows, groups, n, k, type, rng.choice(["bf16", "fp16", "fp32"]), act, rng.random() < 0.3,
                        sources)
    if op == "route":
        tokens, experts = _log_int(rng, 1, 16384), _log_int(rng, 4, 256)
        k = rng.randint(1, min(8, experts))
        return _route("", tokens, experts, k, rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5,
                      rng.randint(0, tokens // 4))
    n = 8 * _log_int(rng, 16, 1024)
    k = rng.randint(1, 8)
    return _combine("", _log_int(rng, 1, max(1, min(16384, 10 ** 8 // (n * k)))), k, n,
                    rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["bf16", "fp16", "fp32"]))


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _blocks(n):
    return -(-n // BLOCK)


def _row_bytes(cols, type):
    """Elements of a row that ends at a multiple of 16 bytes: where the operands' rows have to start."""
    each = 16 // TYPES[type].itemsize
    return -(-cols // each) * each


def _padded(x, ld):
    """x with rows `ld` elements apart."""
    if x.shape[-1] == ld:
        return x.contiguous()
    base = torch.zeros(x.shape[:-1] + (ld,), dtype=x.dtype, device=x.device)
    base[..., :x.shape[-1]].copy_(x)
    return base[..., :x.shape[-1]]


def _stored(x, block_rows):
    """x [..., rows, cols] as e4m3 with one fp32 scale (any, not powers of two alone) for each block."""
    *lead, r, c = x.shape
    rb, cb = -(-r // block_rows), _blocks(c)
    pad = torch.zeros(*lead, rb * block_rows, cb * BLOCK, device=x.device)
    pad[..., :r, :c] = x
    blocks = pad.view(*lead, rb, block_rows, cb, BLOCK)
    scales = (blocks.abs().amax(dim=(-3, -1)) / E4M3_MAX).clamp_min(1e-12)
    q = (blocks / scales[..., :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(*lead, rb * block_rows, cb * BLOCK)
    q = q[..., :r, :c].to(torch.float8_e4m3fn)
    return _padded(q.view(torch.uint8), _row_bytes(c, "e4m3")).view(torch.float8_e4m3fn), scales.contiguous()


def _sizes(rows, groups, seed):
    """Ragged: some groups take several times the mean, some little or nothing."""
    rng = np.random.default_rng(seed)
    return rng.multinomial(rows, rng.dirichlet(np.full(groups, 3.0)))


def _pointer(t):
    return t.data_ptr() if t is not None else None


def prepare(case, seed):
    gen, op = _generator(seed), case["op"]
    s = dict(case)
    if op == "quantise":
        rows, cols = case["rows"], case["cols"]
        sources = case["sources"] or rows
        x = _normal(gen, sources, cols)
        if case["block_rows"] == 1:     # activations: a few channels are much larger than the others
            x *= 1.0 + 15.0 * (torch.rand(cols, generator=gen, device=DEVICE) < 0.01)
        else:
            x *= (2.0 / cols) ** 0.5
        s["x"] = x = x.to(TYPES[case["type"]])
        s["index"] = None
        if case["sources"]:
            s["index"] = (torch.randperm(rows, generator=gen, device=DEVICE) % sources).to(torch.int32)
        ldq = _row_bytes(cols, "e4m3")
        s["q"] = torch.zeros(rows, ldq, dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn)[:, :cols]
        s["scales"] = torch.empty(-(-rows // case["block_rows"]), _blocks(cols), device=DEVICE)
        s["args"] = (x.data_ptr(), CODES[case["type"]], sources, cols, cols, _pointer(s["index"]), rows,
                     case["block_rows"], s["q"].data_ptr(), ldq, s["scales"].data_ptr())
    elif op == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        a = _normal(gen, rows, k)
        if case["act"] == "relu":       # behind another layer of the kind
            a = a.clamp_min_(0)
        s["a"], s["scale_a"] = _stored(a, 1)
        s["b"], s["scale_b"] = _stored(_normal(gen, n, k) * (2.0 / k) ** 0.5, BLOCK)
        s["bias"] = _normal(gen, n) * 0.1 if case["bias"] else None
        s["y"] = torch.empty(rows, n, dtype=TYPES[case["out"]], device=DEVICE)
        s["args"] = (s["a"].data_ptr(), s["a"].stride(0), s["scale_a"].data_ptr(), s["b"].data_ptr(),
                     s["b"].stride(0), s["scale_b"].data_ptr(), _pointer(s["bias"]), rows, n, k, ACTS[case["act"]],
                     s["y"].data_ptr(), CODES[case["out"]], n)
    elif op == "grouped":
        rows, n, k, groups, type = case["rows"], case["n"], case["k"], case["groups"], case["type"]
        both = 2 if case["act"] == "gated" else 1
        sources = case["sources"] or rows
        a, b = _normal(gen, sources, k), _normal(gen, groups * both, n, k) * (2.0 / k) ** 0.5
        s["scale_a"] = s["scale_b"] = None
        if type == "e4m3":
            s["a"], s["scale_a"] = _stored(a, 1)
            s["b"], s["scale_b"] = _stored(b, BLOCK)
        else:
            s["a"], s["b"] = (_padded(t.to(TYPES[type]), _row_bytes(k, type)) for t in (a, b))
        s["bias"] = _normal(gen, groups * both, n) * 0.1 if case["bias"] else None
        sizes = _sizes(rows, groups, seed)
        s["largest"] = int(sizes.max())
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).to(DEVICE)
        s["index"] = None
        if case["sources"]:
            s["index"] = (torch.randperm(rows, generator=gen, device=DEVICE) % sources).to(torch.int32)
        s["y"] = torch.empty(rows, n, dtype=TYPES[case["out"]], device=DEVICE)
        s["args"] = (s["a"].data_ptr(), CODES[type], sources, s["a"].stride(0), _pointer(s["scale_a"]),
                     _pointer(s["index"]), s["offsets"].data_ptr(), groups, s["b"].data_ptr(), s["b"].stride(-2),
                     _pointer(s["scale_b"]), _pointer(s["bias"]), rows, n, k, ACTS[case["act"]], s["y"].data_ptr(),
                     CODES[case["out"]], n)
    elif op == "route":
        tokens, experts, k = case["tokens"], case["experts"], case["k"]
        logits = _normal(gen, tokens, experts) * 2.0
        logits[tokens - case["padded"]:] = -math.inf     # the batch's padding goes nowhere
        s["logits"] = logits = logits.to(TYPES[case["type"]])
        whole = {"dtype": torch.int32, "device": DEVICE}
        s["chosen"], s["position"] = torch.empty(tokens, k, **whole), torch.empty(tokens, k, **whole)
        s["weights"] = torch.empty(tokens, k, device=DEVICE)
        s["offsets"], s["order"] = torch.empty(experts + 1, **whole), torch.empty(tokens * k, **whole)
        # counts of each expert for each 32 tokens, and room to align them
        s["work"] = torch.empty(4 * (experts + 32) * (_blocks(4 * tokens) + 2), dtype=torch.uint8, device=DEVICE)
        s["args"] = (logits.data_ptr(), CODES[case["type"]], tokens, experts, experts, k, int(case["normalise"]),
                     s["chosen"].data_ptr(), s["weights"].data_ptr(), s["offsets"].data_ptr(), s["order"].data_ptr(),
                     s["position"].data_ptr(), s["work"].data_ptr(), s["work"].numel())
    else:
        tokens, k, n = case["tokens"], case["k"], case["n"]
        rows = tokens * k
        s["y"] = _normal(gen, rows, n).to(TYPES[case["type"]])
        s["position"] = torch.randperm(rows, generator=gen, device=DEVICE).to(torch.int32).view(tokens, k)
        s["weights"] = torch.softmax(_normal(gen, tokens, k), dim=1)
        s["out_rows"] = torch.empty(tokens, n, dtype=TYPES[case["out"]], device=DEVICE)
        s["args"] = (s["y"].data_ptr(), CODES[case["type"]], rows, n, s["position"].data_ptr(),
                     s["weights"].data_ptr(), tokens, k, n, s["out_rows"].data_ptr(), CODES[case["out"]], n)
    return s


# ---------------------------------------------------------------------------------------------- plain form
def _activation(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "none":
        return v
    if act == "tanh":
        return 1.0 - 2.0 / (1.0 + torch.exp(2.0 * v))
    s = 1.0 / (1.0 + torch.exp(-v))
    return s if act == "sigmoid" else v * s


def _values(q, scales, block_rows):
    """The fp32 numbers that e4m3 rows and their scales stand for."""
    r, c = q.shape[-2:]
    scales = scales.repeat_interleave(BLOCK, -1)[..., :c]
    if block_rows > 1:
        scales = scales.repeat_interleave(block_rows, -2)[..., :r, :]
    return q.float() * scales


def _plain_quantise(s):
    x = s["x"]
    if s["index"] is not None:
        x = x[s["index"].long()]
    r, c = x.shape
    br = s["block_rows"]
    rb, cb = -(-r // br), _blocks(c)
    x = torch.nn.functional.pad(x.float(), (0, cb * BLOCK - c, 0, rb * br - r)).view(rb, br, cb, BLOCK)
    amax = x.abs().amax(dim=(1, 3))
    # the smallest power of two with amax / scale <= 448: 448 = 1.75 * 2^8
    mantissa, exponent = torch.frexp(amax)       # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > 0.875).int()
    scales = torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, -126)).clamp_min(-126))
    q = (x / scales[:, None, :, None]).view(rb * br, cb * BLOCK)[:r, :c].to(torch.float8_e4m3fn)
    return {"q": q, "scales": scales}


def _plain_product(s):
    y = _values(s["a"], s["scale_a"], 1) @ _values(s["b"], s["scale_b"], BLOCK).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return _activation(y, s["act"]).to(TYPES[s["out"]])


def _plain_grouped(s):
    """Every group padded to the largest one's rows, one batched product."""
    a, b, groups, rows = s["a"], s["b"], s["groups"], s["rows"]
    if s["type"] == "e4m3":
        a, b = _values(a, s["scale_a"], 1), _values(b, s["scale_b"], BLOCK)
    else:
        a, b = a.float(), b.float()
    slot = torch.arange(rows, device=DEVICE)
    if s["index"] is not None:
        a = a[s["index"].long()]
    offsets = s["offsets"].long()
    group = (slot[:, None] >= offsets[None, 1:]).sum(1)
    within = slot - offsets[group]
    room = torch.zeros(groups, max(1, s["largest"]), s["k"], device=DEVICE)
    room[group, within] = a
    b = b.reshape(groups, -1, s["k"])
    y = torch.bmm(room, b.transpose(1, 2))[group, within]
    if s["bias"] is not None:
        y = y + s["bias"].view(groups, -1)[group]
    if s["act"] == "gated":
        y = _activation(y[:, :s["n"]], "silu") * y[:, s["n"]:]
    else:
        y = _activation(y, s["act"])
    return y.to(TYPES[s["out"]])


def _plain_route(s):
    tokens, experts, k = s["tokens"], s["experts"], s["k"]
    logits = s["logits"].float()
    high, at = torch.sort(logits, dim=1, descending=True, stable=True)
    high, at = high[:, :k], at[:, :k]
    taken = high > -math.inf
    some = taken[:, :1]
    top = torch.where(some, high[:, :1], torch.zeros_like(high[:, :1]))
    e = torch.exp(high - top)
    total = (e if s["normalise"] else torch.exp(logits - top)).sum(1, keepdim=True)
    weights = torch.where(taken, e / torch.where(some, total, torch.ones_like(total)), torch.zeros_like(e))
    chosen = torch.where(taken, at, torch.full_like(at, -1)).int()
    flat = torch.where(taken, at, torch.full_like(at, experts)).view(-1)
    ordered, slots = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(experts + 1, device=DEVICE))
    used = ordered < experts
    order = torch.where(used, slots // k, torch.full_like(slots, -1))
    position = torch.empty_like(slots)
    position[slots] = torch.where(used, torch.arange(tokens * k, device=DEVICE), torch.full_like(slots, -1))
    return {"chosen": chosen, "weights": weights, "offsets": offsets.int(), "order": order.int(),
            "position": position.int().view(tokens, k)}


def _plain_combine(s):
    rows = s["y"][s["position"].long()].float()
    return (rows * s["weights"][:, :, None]).sum(1).to(TYPES[s["out"]])


PLAIN = {"quantise": _plain_quantise, "product": _plain_product, "grouped": _plain_grouped, "route": _plain_route,
         "combine": _plain_combine}


# ---------------------------------------------------------------------------------------------- the runtime's
ENTRY = {"quantise": "occamy_quantize_e4m3", "product": "occamy_matmul_e4m3", "grouped": "occamy_matmul_grouped",
         "route": "occamy_route_experts", "combine": "occamy_combine_experts"}
_entries = {}


def _entry(op):
    if op not in _entries:
        from occamy_b200 import runtime
        _entries[op] = getattr(runtime.lib(), ENTRY[op])
    return _entries[op]


def run(state):
    op = state["op"]
    if not own:
        return PLAIN[op](state)
    code = _entry(op)(*state["args"], torch.cuda.current_stream().cuda_stream)
    if code:
        raise RuntimeError(f"{ENTRY[op]}: {code}")
    if op == "quantise":
        return {"q": state["q"], "scales": state["scales"]}
    if op == "route":
        return {name: state[name] for name in ("chosen", "weights", "offsets", "order", "position")}
    return state["out_rows"] if op == "combine" else state["y"]


# ---------------------------------------------------------------------------------------------- work, 64 bits
def work(case):
    """Inputs read once, outputs written once; multiply-adds count as two operations."""
    size = {t: TYPES[t].itemsize for t in TYPES}
    op = case["op"]
    if op == "quantise":
        rows, cols = case["rows"], case["cols"]
        blocks = -(-rows // case["block_rows"]) * _blocks(cols)
        index = 4 * rows if case["sources"] else 0
        return {"bytes": (case["sources"] or rows) * cols * size[case["type"]] + rows * cols + 4 * blocks + index,
                "flops": 2 * rows * cols}
    if op == "product":
        rows, n, k = case["rows"], case["n"], case["k"]
        scales = 4 * (rows + _blocks(n)) * _blocks(k)
        return {"bytes": rows * k + n * k + scales + rows * n * size[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    if op == "grouped":
        rows, n, k, groups = case["rows"], case["n"], case["k"], case["groups"]
        both = 2 if case["act"] == "gated" else 1
        live = groups * (1.0 - (1.0 - 1.0 / groups) ** rows)     # groups that have rows, if all are alike
        e = size[case["type"]]
        scales = 4 * ((case["sources"] or rows) + both * live * _blocks(n)) * _blocks(k) if e == 1 else 0
        return {"bytes": (case["sources"] or rows) * k * e + live * both * n * k * e + scales
                + rows * n * size[case["out"]], "flops": 2 * rows * n * both * k}
    if op == "route":
        tokens, experts, k = case["tokens"], case["experts"], case["k"]
        return {"bytes": tokens * experts * size[case["type"]] + 16 * tokens * k + 4 * experts,
                "flops": 3 * tokens * experts}
    tokens, k, n = case["tokens"], case["k"], case["n"]
    return {"bytes": tokens * k * n * size[case["type"]] + tokens * n * size[case["out"]] + 8 * tokens * k,
            "flops": 2 * tokens * k * n}


def _exact_activation(v, act):
    if act == "relu":
        return v.clamp(min=0)
    return {"none": lambda t: t, "tanh": torch.tanh, "sigmoid": torch.sigmoid,
            "silu": lambda t: t * torch.sigmoid(t)}[act](v)


def _exact_matrix(q, scales, high):
    """[rows, cols] in 64 bits: blocks of `high` x 128 times their scale."""
    out = q.double()
    for i in range(scales.shape[1]):
        part = out[:, i * BLOCK:(i + 1) * BLOCK]
        part *= scales[:, i].double().repeat_interleave(high)[:out.shape[0], None]
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantise":
        x = s["x"].double()
        if s["index"] is not None:
            x = x.index_select(0, s["index"].long())
        r, c = x.shape
        br = case["block_rows"]
        q = torch.empty(r, c, dtype=torch.float64, device=DEVICE)
        scales = torch.empty(-(-r // br), _blocks(c), dtype=torch.float64, device=DEVICE)
        for j in range(_blocks(c)):
            part = x[:, j * BLOCK:(j + 1) * BLOCK]
            if br > 1:
                top = torch.stack([p.abs().max() for p in part.split(br)])
            else:
                top = part.abs().amax(1)
            scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp(min=-126))
            scale = torch.where(scale * E4M3_MAX < top, scale * 2, scale)                  # the logarithm's rounding
            scale = torch.where((scale * (E4M3_MAX / 2) >= top) & (scale > 2.0 ** -126), scale / 2, scale)
            v = part / scale.repeat_interleave(br)[:r, None]
            # e4m3: four significant bits down to 2^-6, then steps of 2^-9; ties to even
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
            q[:, j * BLOCK:(j + 1) * BLOCK] = torch.round(v / step) * step
            scales[:, j] = scale
        return {"q": q, "scales": scales}
    if op == "product":
        y = _exact_matrix(s["a"], s["scale_a"], 1) @ _exact_matrix(s["b"], s["scale_b"], BLOCK).T
        return _exact_activation(y + (s["bias"].double() if s["bias"] is not None else 0.0), case["act"])
    if op == "grouped":
        n, both = case["n"], 2 if case["act"] == "gated" else 1
        a = _exact_matrix(s["a"], s["scale_a"], 1) if s["scale_a"] is not None else s["a"].double()
        y = torch.empty(case["rows"], n, dtype=torch.float64, device=DEVICE)
        offsets = s["offsets"].tolist()
        for g in range(case["groups"]):
            lo, hi = offsets[g], offsets[g + 1]
            if lo == hi:
                continue
            rows = a[s["index"][lo:hi].long()] if s["index"] is not None else a[lo:hi]
            parts = []
            for m in range(g * both, g * both + both):
                b = _exact_matrix(s["b"][m], s["scale_b"][m], BLOCK) if s["scale_b"] is not None else s["b"][m].double()
                parts.append(rows @ b.T + (s["bias"][m].double() if s["bias"] is not None else 0.0))
            y[lo:hi] = _exact_activation(parts[0], "silu") * parts[1] if both == 2 else \
                _exact_activation(parts[0], case["act"])
        return y
    if op == "route":
        logits = s["logits"].double().cpu().numpy()
        tokens, experts, k = case["tokens"], case["experts"], case["k"]
        at = np.argsort(-logits, axis=1, kind="stable")[:, :k]
        high = np.take_along_axis(logits, at, 1)
        live = tokens - case["padded"]
        weights = np.zeros((tokens, k))
        e = np.exp(high[:live] - high[:live, :1])
        total = e if case["normalise"] else np.exp(logits[:live] - high[:live, :1])
        weights[:live] = e / total.sum(1, keepdims=True)
        at[live:] = -1
        of_expert = [[] for _ in range(experts)]
        for t in range(live):
            for j in range(k):
                of_expert[at[t, j]].append(t * k + j)
        offsets = np.cumsum([0] + [len(v) for v in of_expert])
        slots = np.array([v for each in of_expert for v in each], dtype=np.int64)
        order, position = np.full(tokens * k, -1), np.full(tokens * k, -1)
        order[:len(slots)] = slots // k
        position[slots] = np.arange(len(slots))

        def whole(v):
            return torch.from_numpy(v.astype(np.int32))
        return {"chosen": whole(at), "weights": torch.from_numpy(weights), "offsets": whole(offsets),
                "order": whole(order), "position": whole(position.reshape(tokens, k))}
    out = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device=DEVICE)
    for j in range(case["k"]):
        out += s["y"].double().index_select(0, s["position"][:, j].long()) * s["weights"][:, j, None].double()
    return out
