"""The 8-bit and grouped operators on torch tensors, and what they compute in 64 bits."""
import torch

from occamy_b200 import runtime as rt

CODE = {torch.float32: rt.F32, torch.bfloat16: rt.BF16, torch.float16: rt.F16, torch.float8_e4m3fn: rt.E4M3}
ACT = {"sigmoid": 0, "relu": 1, "tanh": 2, "clip": 3, "none": 5, "silu": 6, "gated": 7}
E4M3_MAX = 448.0


def ptr(t):
    return None if t is None else t.data_ptr()


def stream_of(stream):
    return torch.cuda.current_stream().cuda_stream if stream is None else stream


def blocks(n):
    return -(-n // 128)


def quantize(x, q, scales, block_rows=1, index=None, stream=None):
    return rt.lib().occamy_quantize_e4m3(ptr(x), CODE[x.dtype], x.shape[0], x.shape[1], x.stride(0), ptr(index),
                                         q.shape[0], block_rows, ptr(q), q.stride(0), ptr(scales), stream_of(stream))


def matmul(a, scale_a, b, scale_b, out, act="none", bias=None, stream=None):
    return rt.lib().occamy_matmul_e4m3(ptr(a), a.stride(0), ptr(scale_a), ptr(b), b.stride(0), ptr(scale_b), ptr(bias),
                                       out.shape[0], out.shape[1], a.shape[1], ACT[act], ptr(out), CODE[out.dtype],
                                       out.stride(0), stream_of(stream))


def grouped(a, offsets, b, out, scale_a=None, scale_b=None, act="none", bias=None, index=None, stream=None):
    """b: [groups (, 2), N, K]."""
    return rt.lib().occamy_matmul_grouped(ptr(a), CODE[a.dtype], a.shape[0], a.stride(0), ptr(scale_a), ptr(index),
                                          ptr(offsets), b.shape[0], ptr(b), b.stride(-2), ptr(scale_b), ptr(bias),
                                          out.shape[0], out.shape[1], a.shape[1], ACT[act], ptr(out), CODE[out.dtype],
                                          out.stride(0), stream_of(stream))


def route(logits, k, normalise, stream=None, workspace=None):
    """(code, chosen, weights, offsets, order, position); results start out as 77."""
    tokens, experts = logits.shape

    def whole(*shape):
        return torch.full(shape, 77, dtype=torch.int32, device=logits.device)
    chosen, offsets, order, position = whole(tokens, k), whole(experts + 1), whole(tokens * k), whole(tokens, k)
    weights = torch.full((tokens, k), 77.0, device=logits.device)
    if workspace is None:
        need = rt.lib().occamy_route_experts_workspace(tokens, experts, k)
        workspace = torch.empty(max(need, 4), dtype=torch.uint8, device=logits.device)
    code = rt.lib().occamy_route_experts(ptr(logits), CODE[logits.dtype], tokens, experts, logits.stride(0), k,
                                         int(normalise), ptr(chosen), ptr(weights), ptr(offsets), ptr(order),
                                         ptr(position), ptr(workspace), workspace.numel(), stream_of(stream))
    return code, chosen, weights, offsets, order, position


def combine(y, position, weights, out, stream=None):
    return rt.lib().occamy_combine_experts(ptr(y), CODE[y.dtype], y.shape[0], y.stride(0), ptr(position), ptr(weights),
                                           out.shape[0], position.shape[1], out.shape[1], ptr(out), CODE[out.dtype],
                                           out.stride(0), stream_of(stream))


# ------------------------------------------------------------------------------------------- operands
def rows_apart(x, multiple, fill=None):
    """x with rows a multiple of `multiple` elements apart, one more than needed; what is between holds `fill`."""
    ld = (-(-x.shape[-1] // multiple) + 1) * multiple
    base = torch.empty(x.shape[:-1] + (ld,), dtype=x.dtype, device=x.device)
    if x.element_size() == 1:
        base.view(torch.uint8).fill_(0x7f)      # NaN
    else:
        base.fill_(float("nan") if fill is None else fill)
    view = base[..., :x.shape[-1]]
    view.copy_(x)
    return view


def e4m3(gen, *shape, scale=1.0, block_rows=1):
    """Random e4m3 values whose rows have NaN between them, and fp32 scales (no powers of two)."""
    x = (torch.randn(shape, generator=gen, device="cuda") * 40).clamp(-E4M3_MAX, E4M3_MAX)
    q = rows_apart(x.to(torch.float8_e4m3fn).view(torch.uint8), 16).view(torch.float8_e4m3fn)
    r = -(-shape[-2] // block_rows)
    s = (torch.rand(shape[:-2] + (r, blocks(shape[-1])), generator=gen, device="cuda") + 0.5) * (scale / 40)
    return q, s


def values(q, scales, block_rows):
    """In 64 bits."""
    s = scales.double().repeat_interleave(128, -1)[..., :q.shape[-1]]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, -2)[..., :q.shape[-2], :]
    return q.float().double() * s


def activation(v, act):
    return {"none": lambda: v, "relu": lambda: v.clamp(min=0), "tanh": lambda: torch.tanh(v),
            "sigmoid": lambda: torch.sigmoid(v), "clip": lambda: v.clamp(0, 6),
            "silu": lambda: v * torch.sigmoid(v)}[act]()


def product64(a, b, bias, act, out_type):
    """(result, how far a kernel may be off) of rows a [M, K] and weights b [N, K] or [2, N, K], in 64 bits.

    The products of two e4m3, bf16 or fp16 numbers are exact in fp32.  A tensor instruction adds 16 or 32 of them to
    a running sum; each such addition, and each scaled block's, is taken to be off by at most 2^-22 of the sum of the
    magnitudes so far (two bits short of fp32's own rounding: the unit aligns its summands to the largest before
    it adds).  Scaling a block rounds twice more, the bias once.  Activations have slopes of at most 1.1 and are
    computed within 8 units of the last place.  The result is rounded once."""
    both = b if b.dim() == 3 else b[None]
    v, off = [], []
    for h in range(both.shape[0]):
        r = a @ both[h].T
        size = a.abs() @ both[h].abs().T
        if bias is not None:
            r, size = r + bias.double().view(both.shape[0], -1)[h], size + bias.double().abs().view(both.shape[0], -1)[h]
        v.append(r)
        off.append((a.shape[1] / 16 + 2 * blocks(a.shape[1]) + 4) * 2.0 ** -22 * size)
    if len(v) == 2:
        g = activation(v[0], "silu")
        y = g * v[1]
        slack = 1.1 * off[0] * (v[1].abs() + off[1]) + (g.abs() + 1.1 * off[0]) * off[1] + 16 * 2.0 ** -24 * y.abs()
    else:
        y = activation(v[0], act)
        slack = 1.1 * off[0] + 8 * 2.0 ** -24 * y.abs()
    info = torch.finfo(out_type)
    return y, slack + (y.abs() + slack) * (info.eps / 2) + info.tiny * info.eps


def close(got, want, slack):
    got = got.double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - slack).max().item() if got.numel() else 0.0
    assert worst <= 0, worst
