"""Every form that the products have, for each kind of operands: the counters say that the call took it."""
import itertools
import math

import pytest
import torch

import expert_calls as ec
from occamy_b200 import runtime as rt
from test_gpu_expert_ops import KEEP, TYPES, generator, kept, no_errors  # noqa: F401

pytestmark = pytest.mark.gpu

# (operands, gated, rows chosen by an index, rows of a tile, CTAs that share its K, rows, groups, N, K); on 148 SMs
CASES = [
    ("16", 0, 0, 32, 1, 104, 3, 144, 80), ("16", 0, 0, 32, 2, 953, 9, 144, 1000),
    ("16", 0, 0, 32, 4, 109, 3, 136, 1192), ("16", 0, 0, 32, 8, 105, 3, 152, 2192),
    ("16", 0, 0, 64, 1, 3034, 40, 400, 80), ("16", 0, 0, 64, 2, 1047, 9, 264, 1176),
    ("16", 0, 0, 64, 4, 1143, 6, 168, 1112), ("16", 0, 0, 64, 8, 519, 6, 144, 2008),
    ("16", 0, 0, 256, 1, 830, 3, 160, 520), ("16", 0, 1, 32, 1, 104, 3, 144, 80),
    ("16", 0, 1, 32, 2, 117, 3, 136, 464), ("16", 0, 1, 32, 4, 109, 3, 136, 1192),
    ("16", 0, 1, 32, 8, 105, 3, 152, 2192), ("16", 0, 1, 64, 1, 2862, 40, 296, 80),
    ("16", 0, 1, 64, 2, 1441, 9, 272, 464), ("16", 0, 1, 64, 4, 1093, 6, 176, 976),
    ("16", 0, 1, 64, 8, 519, 6, 144, 2008), ("16", 1, 0, 32, 1, 141, 3, 72, 88),
    ("16", 1, 0, 32, 2, 360, 9, 216, 976), ("16", 1, 0, 32, 4, 100, 3, 96, 1288),
    ("16", 1, 0, 32, 8, 110, 3, 80, 2088), ("16", 1, 0, 64, 1, 421, 6, 1352, 80),
    ("16", 1, 0, 64, 2, 745, 9, 216, 1136), ("16", 1, 0, 64, 4, 1051, 9, 80, 1296),
    ("16", 1, 0, 64, 8, 497, 6, 72, 2488), ("16", 1, 0, 256, 1, 2292, 6, 216, 80),
    ("16", 1, 1, 32, 1, 141, 3, 72, 88), ("16", 1, 1, 32, 2, 110, 3, 112, 464),
    ("16", 1, 1, 32, 4, 100, 3, 96, 1288), ("16", 1, 1, 32, 8, 110, 3, 80, 2088),
    ("16", 1, 1, 64, 1, 2243, 24, 208, 80), ("16", 1, 1, 64, 2, 464, 6, 328, 976),
    ("16", 1, 1, 64, 4, 1282, 9, 80, 968), ("16", 1, 1, 64, 8, 497, 6, 72, 2488),
    ("e4m3", 0, 0, 32, 1, 127, 3, 144, 152), ("e4m3", 0, 0, 32, 2, 109, 3, 136, 1192),
    ("e4m3", 0, 0, 32, 4, 105, 3, 152, 2192), ("e4m3", 0, 0, 64, 1, 825, 40, 800, 152),
    ("e4m3", 0, 0, 64, 2, 472, 6, 664, 1968), ("e4m3", 0, 0, 64, 4, 620, 9, 408, 2280),
    ("e4m3", 0, 0, 128, 1, 2250, 9, 392, 152), ("e4m3", 0, 0, 128, 2, 1446, 9, 160, 1944),
    ("e4m3", 0, 0, 128, 4, 1361, 3, 136, 2152), ("e4m3", 0, 0, 256, 1, 980, 3, 280, 968),
    ("e4m3", 0, 1, 32, 1, 127, 3, 144, 152), ("e4m3", 0, 1, 32, 2, 109, 3, 136, 1192),
    ("e4m3", 0, 1, 32, 4, 105, 3, 152, 2192), ("e4m3", 0, 1, 64, 1, 825, 40, 800, 152),
    ("e4m3", 0, 1, 64, 2, 472, 6, 664, 1968), ("e4m3", 0, 1, 64, 4, 620, 9, 408, 2280),
    ("e4m3", 0, 1, 128, 1, 2250, 9, 392, 152), ("e4m3", 0, 1, 128, 2, 1446, 9, 160, 1944),
    ("e4m3", 0, 1, 128, 4, 1361, 3, 136, 2152), ("e4m3", 0, 1, 256, 1, 980, 3, 280, 968),
    ("e4m3", 1, 0, 32, 1, 97, 3, 72, 184), ("e4m3", 1, 0, 32, 2, 100, 3, 96, 1288),
    ("e4m3", 1, 0, 32, 4, 98, 3, 80, 1984), ("e4m3", 1, 0, 64, 1, 740, 40, 424, 152),
    ("e4m3", 1, 0, 64, 2, 806, 9, 200, 1992), ("e4m3", 1, 0, 64, 4, 346, 3, 520, 1968),
    ("e4m3", 1, 0, 128, 1, 2417, 6, 208, 152), ("e4m3", 1, 0, 128, 2, 1465, 9, 72, 2648),
    ("e4m3", 1, 0, 128, 4, 1170, 3, 80, 2120), ("e4m3", 1, 0, 256, 1, 817, 3, 136, 1120),
    ("e4m3", 1, 1, 32, 1, 97, 3, 72, 184), ("e4m3", 1, 1, 32, 2, 100, 3, 96, 1288),
    ("e4m3", 1, 1, 32, 4, 98, 3, 80, 1984), ("e4m3", 1, 1, 64, 1, 740, 40, 424, 152),
    ("e4m3", 1, 1, 64, 2, 806, 9, 200, 1992), ("e4m3", 1, 1, 64, 4, 346, 3, 520, 1968),
    ("e4m3", 1, 1, 128, 1, 2417, 6, 208, 152), ("e4m3", 1, 1, 128, 2, 1465, 9, 72, 2648),
    ("e4m3", 1, 1, 128, 4, 1170, 3, 80, 2120), ("e4m3", 1, 1, 256, 1, 817, 3, 136, 1120),
]


def split(rows, groups):
    """Sizes of groups: one empty, one row, the others unequal."""
    if groups == 1:
        return [rows]
    some = [1 + 2 * (g % 3) for g in range(groups)]
    some[1] = 0
    left = rows - 1
    sizes = [left * s // sum(some[:-1]) for s in some[:-1]] + [1]
    sizes[0] += rows - sum(sizes)
    return sizes


class Problem:
    """Operands of one grouped product, and its result in 64 bits."""

    def __init__(self, type, gated, indexed, rows, groups, n, k, seed=0):
        gen = generator(seed)
        self.sizes, self.n, self.gated = split(rows, groups), n, gated
        both = (2,) if gated else ()
        sources = max(3, rows // 2) if indexed else rows
        self.sa = self.sb = self.index = None
        if type == "e4m3":
            self.a, self.sa = ec.e4m3(gen, sources, k)
            self.b, self.sb = ec.e4m3(gen, groups, *both, n, k, scale=k ** -0.5, block_rows=128)
        else:
            t = TYPES[["bf16", "fp16"][seed % 2]]
            self.a = ec.rows_apart(torch.randn(sources, k, generator=gen, device="cuda").to(t), 8)
            self.b = ec.rows_apart((torch.randn(groups, *both, n, k, generator=gen, device="cuda") * k ** -0.5).to(t), 8)
        self.bias = torch.randn(groups, *both, n, generator=gen, device="cuda") if seed % 3 else None
        if indexed:
            self.index = torch.randint(-1, sources + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        self.offsets = torch.tensor(list(itertools.accumulate([0] + self.sizes)), dtype=torch.int32, device="cuda")

    def __call__(self, out, act):
        return ec.grouped(self.a, self.offsets, self.b, out, self.sa, self.sb, act, self.bias, self.index)

    def check(self, out, act):
        a = ec.values(self.a, self.sa, 1) if self.sa is not None else self.a.double()
        if self.index is not None:
            there = (self.index >= 0) & (self.index < a.shape[0])
            a = torch.where(there[:, None], a[self.index.long().clamp(0, a.shape[0] - 1)], torch.zeros_like(a[:1]))
        lo = 0
        for g, size in enumerate(self.sizes):
            if size:
                b = ec.values(self.b[g], self.sb[g], 128) if self.sb is not None else self.b[g].double()
                ec.close(out[lo:lo + size], *ec.product64(a[lo:lo + size], b, self.bias[g] if self.bias is not None else None,
                                                          act, out.dtype))
            lo += size


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_form(case):
    type, gated, indexed, tile, shares, rows, groups, n, k = case
    seed = CASES.index(case)
    p = Problem(type, gated, indexed, rows, groups, n, k, seed)
    act = "gated" if gated else ["none", "relu", "silu"][seed % 3]
    out_type = list(TYPES.values())[seed % 3]
    for extra in (8, 3):       # rows of the result at multiples of 16 bytes, and anywhere
        base, out = kept(rows, n, out_type, extra=extra)
        before, shared = rt.form_counters(), rt.products_with_shared_k()
        assert p(out, act) == 0
        assert [f for f, v in rt.form_counters().items() if v != before[f]] == [f"product_{tile}"]
        assert rt.products_with_shared_k() - shared == (shares > 1)
        p.check(out, act)
        assert (base[:, n:].float() == torch.tensor(KEEP).to(out_type).float().item()).all()
        again = torch.full_like(base, KEEP)[:, :n]
        assert p(again, act) == 0
        assert torch.equal(out, again)


@pytest.mark.parametrize("gated,n,indexed,tile", [(False, 1000, False, 32), (True, 512, False, 32), (False, 1096, True, 64)])
def test_1100_rows_of_one_group(gated, n, indexed, tile):
    """The forms of the calls with 1100 rows in test_heights_of_tiles."""
    p = Problem("16", gated, indexed, 1100, 1, n, 328)
    before = rt.form_counters()
    _, out = kept(1100, n, torch.float32)
    act = "gated" if gated else "none"
    assert p(out, act) == 0
    assert [f for f, v in rt.form_counters().items() if v != before[f]] == [f"product_{tile}"]
    p.check(out, act)


@pytest.mark.parametrize("case", [c for c in CASES if c[0] == "e4m3"], ids=lambda c: "-".join(map(str, c[1:])))
def test_scales_whose_product_fp32_does_not_hold(case):
    """Blocks of K in turn with weights' scales of about 1, 2^-75 and 2^64; rows of six kinds:
    0  scales that make up for those
    1  2^-75 where the weights have it: the product is 2^-150, the result about 2^-130; nothing elsewhere
    2  2^64 where the weights have it and 2^-9 once there: the product is 2^128, the result up to 2^127; nothing elsewhere
    3  2^64 where the weights have it, on zeros
    4  nothing, with the smallest scale that quantising gives
    5  of both signs: kinds 0 and 1 in one row, whose small blocks vanish beside the others
    Gated: the gate is about 1/2, what it multiplies is as above."""
    _, gated, indexed, tile, shares, rows, groups, n, k = case
    p = Problem("e4m3", gated, indexed, rows, groups, n, k, 7 + CASES.index(case))
    gen = generator(k)
    blocks = ec.blocks(k)
    e = torch.tensor([0, -75, 64], device="cuda").repeat(blocks)[:blocks]
    p.sb = 0.25 + 0.25 * torch.rand(p.sb.shape, generator=gen, device="cuda")
    if gated:
        p.sb[:, 0] *= torch.exp2(torch.where(e == 64, -64, 0).float())
        p.sb[:, 1] *= torch.exp2(e.float())
        p.bias = torch.zeros(groups, 2, n, device="cuda")
        p.bias[:, 0] = 0.5
    else:
        p.sb *= torch.exp2(e.float())
        p.bias = None
    kind = torch.arange(p.a.shape[0], device="cuda") % 6
    if blocks < 3:
        kind[kind == 2] = 0
    of_kind = torch.stack([-e, torch.where(e == -75, -75, -64), torch.where(e == 64, 64, 0), torch.where(e == 64, 64, -64),
                           torch.full_like(e, -126), torch.where(e == 64, -64, e)])[kind]
    p.sa = torch.exp2(of_kind.float())
    p.sa[kind == 5] *= -1
    along = e.repeat_interleave(128)[:k]
    a = p.a.float()
    a[(kind == 1)[:, None] & (along != -75)] = 0
    a[(kind == 2)[:, None].expand_as(a)] = 0
    if blocks >= 3:
        a[kind == 2, 2 * 128 + 5] = 2.0 ** -9
    a[(kind == 3)[:, None] & (along == 64)] = 0
    a[(kind == 4)[:, None].expand_as(a)] = 0
    p.a = ec.rows_apart(a.to(torch.float8_e4m3fn).view(torch.uint8), 16).view(torch.float8_e4m3fn)
    act = "gated" if gated else "none"
    out = torch.full((rows, n), KEEP, device="cuda")
    before = rt.form_counters()
    assert p(out, act) == 0
    assert [f for f, v in rt.form_counters().items() if v != before[f]] == [f"product_{tile}"]
    p.check(out, act)
    again = torch.empty_like(out)
    assert p(again, act) == 0
    assert torch.equal(out, again)


def test_scales_that_are_no_numbers_or_zero():
    """They act as the formula has it: zero takes its block away, an infinity or NaN makes the sums that it is in NaN or infinite."""
    gen = generator(1)
    (a, sa), (b, sb) = ec.e4m3(gen, 70, 640), ec.e4m3(gen, 200, 640, block_rows=128)
    sa[3, 1], sa[9] = 0.0, 0.0
    sa[20, 2], sa[21, 4], sa[22, 0] = math.inf, math.nan, 2.0 ** -149
    out = torch.empty(70, 200, device="cuda")
    assert ec.matmul(a, sa, b, sb, out) == 0
    good = [r for r in range(70) if r not in (20, 21)]
    want, slack = ec.product64(ec.values(a, sa, 1), ec.values(b, sb, 128), None, "none", torch.float32)
    ec.close(out[good], want[good], slack[good])
    assert not torch.isfinite(out[[20, 21]]).any() and torch.isnan(out[21]).all()


def test_the_smallest_scale():
    """2^-126: a factor below it is a multiple of 2^-149, half a step off at most; a block's sum is below 2^25."""
    gen = generator(2)
    for m in (7, 50, 300, 2100):
        (a, sa), (b, sb) = ec.e4m3(gen, m, 640), ec.e4m3(gen, 200, 640, block_rows=128)
        sa[::3] = 2.0 ** -126
        out = torch.empty(m, 200, device="cuda")
        assert ec.matmul(a, sa, b, sb, out) == 0
        want, slack = ec.product64(ec.values(a, sa, 1), ec.values(b, sb, 128), None, "none", torch.float32)
        ec.close(out, want, slack + 5 * 2.0 ** -125)
