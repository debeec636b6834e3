"""The 8-bit and grouped operators against the same formulas in 64 bits."""
import itertools
import math
import threading

import numpy as np
import pytest
import torch

import expert_calls as ec
from occamy_b200 import runtime as rt

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
KEEP = -7.5   # what results hold before a call


@pytest.fixture(autouse=True)
def no_errors(native_libs):
    rt.last_error(clear=True)
    yield
    rt.synchronize()
    assert rt.last_error(clear=True) == 0


def generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def kept(rows, cols, dtype, extra=3):
    """A result whose rows are `extra` elements longer than it, all of it KEEP."""
    base = torch.full((rows, cols + extra), KEEP, device="cuda").to(dtype)
    return base, base[:, :cols]


# ------------------------------------------------------------------------------------------- quantising
def quantize64(x, block_rows):
    """(values of q as fp64 with NaN, scales) by the definition, on the CPU."""
    x = x.double().cpu().numpy()
    rows, cols = x.shape
    br, bc = -(-rows // block_rows), -(-cols // 128)
    q, scales = np.zeros_like(x), np.zeros((br, bc))
    for i in range(br):
        for j in range(bc):
            at = (slice(i * block_rows, min(rows, (i + 1) * block_rows)), slice(j * 128, min(cols, j * 128 + 128)))
            b = x[at]
            fine = np.isfinite(b)
            top = np.abs(b[fine]).max() if fine.any() else 0.0
            e = -126
            while top > 448.0 * 2.0 ** e:
                e += 1
            v = np.where(fine, b, np.nan) / 2.0 ** e
            step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))) - 3)
            q[at] = np.rint(v / step) * step
            scales[i, j] = 2.0 ** e
    return q, scales


def same_values(q, want):
    got = q.float().double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.nan_to_num(got), np.nan_to_num(want))


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (2, 129), (3, 1000), (128, 128), (129, 257), (130, 640), (5, 2048),
                                       (300, 24)])
def test_quantize(type, block_rows, rows, cols):
    gen = generator(rows * 1000 + cols)
    for aligned in (True, False):
        x = torch.randn(rows, cols, generator=gen, device="cuda") * torch.exp(
            4 * torch.randn(rows, 1, generator=gen, device="cuda"))
        if cols > 140:
            x[:, 128:140] = 0
        x = x.clamp(-6e4, 6e4).to(TYPES[type])
        x = ec.rows_apart(x, 16 if aligned else 1)
        base = torch.full((rows, -(-cols // 16) * 16 + (16 if aligned else 1)), 0x55, dtype=torch.uint8, device="cuda")
        q = base[:, :cols].view(torch.float8_e4m3fn)
        sbase = torch.full((-(-rows // block_rows) * ec.blocks(cols) + 4,), KEEP, device="cuda")
        scales = sbase[:-4].view(-1, ec.blocks(cols))
        assert ec.quantize(x, q, scales, block_rows) == 0
        want, s = quantize64(x, block_rows)
        assert np.array_equal(scales.double().cpu().numpy(), s)
        same_values(q, want)
        assert (base[:, cols:] == 0x55).all() and (sbase[-4:] == KEEP).all()


@pytest.mark.parametrize("type", list(TYPES))
def test_quantize_edges_of_the_types(type):
    t = TYPES[type]
    info = torch.finfo(t)
    x = torch.zeros(12, 256, device="cuda")
    x[1, 0] = 448.0          # the scale is 1 up to here ...
    x[2, 3] = 452.0          # ... and 2 above (bf16: 452 is a number)
    x[3, :] = info.max
    x[4, 7] = info.tiny
    x[5, 9] = 448.0 * 2.0 ** -126
    x[6, :128] = torch.arange(128, device="cuda") / 16.0      # ties
    x[7, 100] = math.inf
    x[7, 101] = 3.0
    x[8, 5] = math.nan
    x[8, 6] = -2.0
    x[9, :] = -math.inf
    x[10, 0], x[10, 1] = 448.0, 2.0 ** -10                    # half of the smallest number: to even, 0
    x[11, 0], x[11, 1], x[11, 2] = 448.0, 1.5 * 2.0 ** -9, -0.0
    x = x.to(t)
    for block_rows in (1, 128):
        q = torch.zeros(12, 256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        scales = torch.zeros(-(-12 // block_rows), 2, device="cuda")
        assert ec.quantize(x, q, scales, block_rows) == 0
        want, s = quantize64(x, block_rows)
        assert np.array_equal(scales.double().cpu().numpy(), s)
        same_values(q, want)


@pytest.mark.parametrize("type", [t for t in TYPES if TYPES[t] != torch.float32])
def test_quantize_every_number_of_the_type(type):
    """By magnitude (blocks of neighbours, the subnormal ones among them), mixed, and as signs alternate."""
    every = torch.arange(1 << 16, dtype=torch.int32)
    mixed = every[torch.randperm(1 << 16, generator=torch.Generator().manual_seed(1))]
    signs = torch.stack([every[:1 << 15], every[1 << 15:]], 1)
    x = torch.cat([every.view(-1, 1024), mixed.view(-1, 1024), signs.reshape(-1, 1024)]).to(torch.int16).cuda().view(TYPES[type])
    for block_rows in (1, 128):
        q = torch.zeros(x.shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        scales = torch.zeros(-(-x.shape[0] // block_rows), 8, device="cuda")
        assert ec.quantize(x, q, scales, block_rows) == 0
        want, s = quantize64(x, block_rows)
        assert np.array_equal(scales.double().cpu().numpy(), s)
        same_values(q, want)
        numbers = ~np.isnan(want)
        assert np.array_equal((q.view(torch.uint8).cpu().numpy() >= 128)[numbers], (x < 0).cpu().numpy()[numbers] |
                              ((x == 0) & (x.view(torch.int16) < 0)).cpu().numpy()[numbers])


@pytest.mark.parametrize("cols", [64, 200, 1024])
def test_quantize_gathers_rows(cols):
    gen = generator(cols)
    x = torch.randn(37, cols, generator=gen, device="cuda").bfloat16()
    index = torch.randint(0, 37, (101,), generator=gen, device="cuda", dtype=torch.int32)
    index[4], index[50], index[100], index[7] = -1, 37, -2147483648, 2147483647
    q = torch.full((101, cols), 0x11, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.full((101, ec.blocks(cols)), KEEP, device="cuda")
    assert ec.quantize(x, q, scales, index=index) == 0
    out = [4, 7, 50, 100]
    there = [i for i in range(101) if i not in out]
    want, s = quantize64(x[index.long()[there]], 1)
    assert np.array_equal(scales[there].double().cpu().numpy(), s)
    same_values(q[there], want)
    assert (q.view(torch.uint8)[out] == 0x11).all() and (scales[out] == KEEP).all()


# ------------------------------------------------------------------------------------------- products
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 127, 129, 256, 257, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (64, 300), (200, 127), (129, 1000), (1000, 257), (264, 2064)])
def test_matmul_e4m3(m, n, k):
    gen = generator(m * 7919 + n * 31 + k)
    a, sa = ec.e4m3(gen, m, k)
    b, sb = ec.e4m3(gen, n, k, scale=k ** -0.5, block_rows=128)
    acts = list(ec.ACT)[:-1]
    act = acts[(m + n + k) % len(acts)]
    bias = torch.randn(n, generator=gen, device="cuda") if (m + n) % 2 else None
    for type in TYPES:
        base, out = kept(m, n, TYPES[type], extra=8 if m % 2 else 3)
        assert ec.matmul(a, sa, b, sb, out, act, bias) == 0
        want, slack = ec.product64(ec.values(a, sa, 1), ec.values(b, sb, 128), bias, act, TYPES[type])
        ec.close(out, want, slack)
        assert (base[:, n:].float() == torch.tensor(KEEP).to(TYPES[type]).float().item()).all()


@pytest.mark.parametrize("m,n,k", [(1, 4096, 25088), (64, 4096, 6272), (700, 2048, 1024), (2100, 1032, 520), (5, 16, 25088)])
@pytest.mark.parametrize("type", list(TYPES))
def test_matmul_e4m3_large(m, n, k, type):
    gen = generator(m + n + k)
    a, sa = ec.e4m3(gen, m, k)
    b, sb = ec.e4m3(gen, n, k, scale=k ** -0.5, block_rows=128)
    out = torch.empty(m, n, dtype=TYPES[type], device="cuda")
    assert ec.matmul(a, sa, b, sb, out, "none") == 0
    want, slack = ec.product64(ec.values(a, sa, 1), ec.values(b, sb, 128), None, "none", TYPES[type])
    ec.close(out, want, slack)
    again = torch.empty_like(out)
    assert ec.matmul(a, sa, b, sb, again, "none") == 0
    assert torch.equal(out, again)


def test_matmul_scales_over_the_range_of_fp32():
    gen = generator(3)
    a, sa = ec.e4m3(gen, 40, 512)
    b, sb = ec.e4m3(gen, 136, 512, block_rows=128)
    sa = sa * 2.0 ** 100
    sb = sb * 2.0 ** -110
    out = torch.empty(40, 136, device="cuda")
    assert ec.matmul(a, sa, b, sb, out) == 0
    want, slack = ec.product64(ec.values(a, sa, 1), ec.values(b, sb, 128), None, "none", torch.float32)
    ec.close(out, want, slack)


@pytest.mark.parametrize("rows_of_nan", [[0], [3, 17], [299]])
def test_matmul_nan_stays_in_its_row(rows_of_nan):
    gen = generator(4)
    a, sa = ec.e4m3(gen, 300, 384)
    b, sb = ec.e4m3(gen, 200, 384, block_rows=128)
    for r in rows_of_nan:
        a.view(torch.uint8)[r, 200] = 0x7f
    out = torch.empty(300, 200, device="cuda")
    assert ec.matmul(a, sa, b, sb, out, "relu") == 0
    bad = torch.isnan(out)
    assert bad[rows_of_nan].all() and bad.sum() == len(rows_of_nan) * 200
    # a weight's NaN stays in its column
    a, sa = ec.e4m3(gen, 300, 384)
    b.view(torch.uint8)[77, 383] = 0xff
    assert ec.matmul(a, sa, b, sb, out, "none") == 0
    bad = torch.isnan(out)
    assert bad[:, 77].all() and bad.sum() == 300


SIZES = {"one": [9], "small": [1, 0, 2, 3, 0], "empty": [0, 0, 0], "ragged": [5, 130, 0, 17, 256, 1, 64, 33],
         "large": [0, 700, 3, 257, 0, 128], "many": [i % 3 for i in range(64)], "most": [i % 2 for i in range(1024)]}


@pytest.mark.parametrize("type", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("act", ["none", "silu", "gated", "relu"])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("n,k", [(64, 64), (200, 328), (136, 1000)])
def test_grouped(type, act, sizes, n, k):
    sizes = SIZES[sizes]
    if len(sizes) == 1024:
        n, k = 16, 40
    seed = len(sizes) * 7 + n + k + len(act)
    gen = generator(seed)
    groups, used = len(sizes), sum(sizes)
    both = (2,) if act == "gated" else ()
    gathered, before, behind = seed % 2 == 0, seed % 3, 4
    rows = before + used + behind
    sources = 23 if gathered else rows
    sa = sb = None
    if type == "e4m3":
        a, sa = ec.e4m3(gen, sources, k)
        b, sb = ec.e4m3(gen, groups, *both, n, k, scale=k ** -0.5, block_rows=128)
    else:
        a = ec.rows_apart(torch.randn(sources, k, generator=gen, device="cuda").to(TYPES[type]), 8)
        b = ec.rows_apart((torch.randn(groups, *both, n, k, generator=gen, device="cuda") * k ** -0.5).to(TYPES[type]), 8)
    bias = torch.randn(groups, *both, n, generator=gen, device="cuda") if seed % 5 < 2 else None
    index = None
    if gathered:
        index = torch.randint(0, sources, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        if used > 2:
            index[before], index[before + 2] = -1, sources     # zeros
    offsets = torch.tensor([before + s for s in itertools.accumulate([0] + sizes)], dtype=torch.int32, device="cuda")
    out_type = list(TYPES.values())[seed % 3]
    base, out = kept(rows, n, out_type, extra=[8, 1][seed % 2])
    assert ec.grouped(a, offsets, b, out, sa, sb, act, bias, index) == 0
    av = ec.values(a, sa, 1) if sa is not None else a.double()
    for g in range(groups):
        lo, hi = before + sum(sizes[:g]), before + sum(sizes[:g + 1])
        if lo == hi:
            continue
        bv = ec.values(b[g], sb[g], 128) if sb is not None else b[g].double()
        if index is None:
            ar = av[lo:hi]
        else:
            i = index[lo:hi].long()
            there = (i >= 0) & (i < sources)
            ar = torch.where(there[:, None], av[i.clamp(0, sources - 1)], torch.zeros_like(av[:1]))
        want, slack = ec.product64(ar, bv, bias[g] if bias is not None else None, act, out_type)
        ec.close(out[lo:hi], want, slack)
    keep = torch.tensor(KEEP).to(out_type).float().item()
    assert (base[:, n:].float() == keep).all()
    assert (base[:before].float() == keep).all() and (base[before + used:].float() == keep).all()


@pytest.mark.parametrize("type", ["bf16", "e4m3"])
def test_grouped_offsets_beyond_the_rows_are_cut_off(type):
    gen = generator(11)
    rows, n, k = 50, 72, 144
    if type == "e4m3":
        a, sa = ec.e4m3(gen, rows, k)
        b, sb = ec.e4m3(gen, 4, n, k, block_rows=128)
    else:
        a, b, sa, sb = (torch.randn(rows, k, generator=gen, device="cuda").bfloat16(),
                        torch.randn(4, n, k, generator=gen, device="cuda").bfloat16(), None, None)
    offsets = torch.tensor([-5, 20, 48, 90, 2147483647], dtype=torch.int32, device="cuda")
    _, out = kept(rows, n, torch.float32)
    guard = out.clone()
    assert ec.grouped(a, offsets, b, out, sa, sb) == 0
    av = ec.values(a, sa, 1) if sa is not None else a.double()
    for g, (lo, hi) in enumerate([(0, 20), (20, 48), (48, 50)]):
        bv = ec.values(b[g], sb[g], 128) if sb is not None else b[g].double()
        want, slack = ec.product64(av[lo:hi], bv, None, "none", torch.float32)
        ec.close(out[lo:hi], want, slack)
    del guard


@pytest.mark.parametrize("type", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [70, 3000])
def test_grouped_offsets_that_go_back(type, rows):
    """An offset below an earlier one counts as that one: no row is in two groups, and none outside is written."""
    gen = generator(13)
    n, k, scale = 1032, 144, rows // 70
    offsets = [10 * scale, 40 * scale, 5, 30, 60 * scale, -7, 60 * scale]
    cut, top = [], 0
    for o in offsets:
        top = max(top, min(max(o, 0), rows))
        cut.append(top)
    groups = len(offsets) - 1
    if type == "e4m3":
        a, sa = ec.e4m3(gen, rows, k)
        b, sb = ec.e4m3(gen, groups, n, k, block_rows=128)
    else:
        a, b, sa, sb = (torch.randn(rows, k, generator=gen, device="cuda").bfloat16(),
                        torch.randn(groups, n, k, generator=gen, device="cuda").bfloat16(), None, None)
    base, out = kept(rows, n, torch.float32, extra=8)
    assert ec.grouped(a, torch.tensor(offsets, dtype=torch.int32, device="cuda"), b, out, sa, sb) == 0
    av = ec.values(a, sa, 1) if sa is not None else a.double()
    for g in range(groups):
        lo, hi = cut[g], cut[g + 1]
        if lo < hi:
            bv = ec.values(b[g], sb[g], 128) if sb is not None else b[g].double()
            ec.close(out[lo:hi], *ec.product64(av[lo:hi], bv, None, "none", torch.float32))
    assert (base[:cut[0]] == KEEP).all() and (base[cut[-1]:] == KEEP).all() and (base[:, n:] == KEEP).all()


@pytest.mark.parametrize("type", ["bf16", "fp16", "e4m3"])
def test_grouped_larger(type):
    """Several tiles of every kind: 1 to 1500 rows a group, gated, gathered."""
    gen = generator(12)
    sizes = [1500, 1, 700, 0, 90, 260, 33, 16]
    rows, sources, n, k = sum(sizes), 1024, 520, 1032
    sa = sb = None
    if type == "e4m3":
        a, sa = ec.e4m3(gen, sources, k)
        b, sb = ec.e4m3(gen, len(sizes), 2, n, k, scale=k ** -0.5, block_rows=128)
    else:
        a = torch.randn(sources, k, generator=gen, device="cuda").to(TYPES[type])
        b = (torch.randn(len(sizes), 2, n, k, generator=gen, device="cuda") * k ** -0.5).to(TYPES[type])
    index = torch.randint(0, sources, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    offsets = torch.tensor(list(itertools.accumulate([0] + sizes)), dtype=torch.int32, device="cuda")
    out = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    assert ec.grouped(a, offsets, b, out, sa, sb, "gated", index=index) == 0
    av = ec.values(a, sa, 1) if sa is not None else a.double()
    lo = 0
    for g, s in enumerate(sizes):
        bv = ec.values(b[g], sb[g], 128) if sb is not None else b[g].double()
        want, slack = ec.product64(av[index[lo:lo + s].long()], bv, None, "gated", torch.bfloat16)
        ec.close(out[lo:lo + s], want, slack)
        lo += s
    again = torch.empty_like(out)
    assert ec.grouped(a, offsets, b, again, sa, sb, "gated", index=index) == 0
    assert torch.equal(out, again)


# Sizes that make the calls take each form: tiles of 32, 64, 128 rows, and of 256 (e4m3: 128 rows and 256 weights).
FORMS = {32: ([3, 0, 30, 33, 1], 264, 520), 64: ([60] * 4 + [0, 130, 64, 65, 7] + [50] * 32, 1032, 264),
         128: ([512, 0, 130, 257, 3, 128], 1032, 1288), 256: ([300, 0, 1, 1290, 256, 511, 777, 64], 2056, 328)}


@pytest.mark.parametrize("rows", list(FORMS))
@pytest.mark.parametrize("type", ["bf16", "e4m3"])
@pytest.mark.parametrize("act,out_type,bias", [("gated", "bf16", False), ("gated", "fp32", True), ("none", "fp32", True),
                                               ("relu", "fp16", True), ("silu", "bf16", False), ("none", "bf16", False)])
@pytest.mark.parametrize("gathered", [False, True])
def test_products_in_every_form(rows, type, act, out_type, bias, gathered):
    sizes, n, k = FORMS[rows]
    both = (2,) if act == "gated" else ()
    if act == "gated":
        n //= 2
        n -= n % 8
    gen = generator(rows + k)
    groups, used = len(sizes), sum(sizes)
    sources = 200 if gathered else used
    sa = sb = None
    if type == "e4m3":
        a, sa = ec.e4m3(gen, sources, k)
        b, sb = ec.e4m3(gen, groups, *both, n, k, scale=k ** -0.5, block_rows=128)
    else:
        a = ec.rows_apart(torch.randn(sources, k, generator=gen, device="cuda").bfloat16(), 8)
        b = ec.rows_apart((torch.randn(groups, *both, n, k, generator=gen, device="cuda") * k ** -0.5).bfloat16(), 8)
    bias = torch.randn(groups, *both, n, generator=gen, device="cuda") if bias else None
    index = None
    if gathered:
        index = torch.randint(0, sources, (used,), generator=gen, device="cuda", dtype=torch.int32)
        index[5], index[used // 2], index[used - 1] = -1, sources, 2147483647
    offsets = torch.tensor(list(itertools.accumulate([0] + sizes)), dtype=torch.int32, device="cuda")
    av = ec.values(a, sa, 1) if sa is not None else a.double()
    for extra in (8, 3):       # rows of the result at multiples of 16 bytes, and anywhere
        base, out = kept(used, n, TYPES[out_type], extra=extra)
        assert ec.grouped(a, offsets, b, out, sa, sb, act, bias, index) == 0
        for g in range(groups):
            lo, hi = sum(sizes[:g]), sum(sizes[:g + 1])
            if lo == hi:
                continue
            bv = ec.values(b[g], sb[g], 128) if sb is not None else b[g].double()
            ar = av[lo:hi]
            if gathered:
                i = index[lo:hi].long()
                there = (i >= 0) & (i < sources)
                ar = torch.where(there[:, None], av[i.clamp(0, sources - 1)], torch.zeros_like(av[:1]))
            ec.close(out[lo:hi], *ec.product64(ar, bv, bias[g] if bias is not None else None, act, TYPES[out_type]))
        assert (base[:, n:].float() == torch.tensor(KEEP).to(TYPES[out_type]).float().item()).all()
        again = torch.full_like(base, KEEP)[:, :n]
        assert ec.grouped(a, offsets, b, again, sa, sb, act, bias, index) == 0
        assert torch.equal(out, again)


@pytest.mark.parametrize("sizes", [[5003, 0, 0, 0, 0, 0, 0, 0], [0, 700, 600, 650, 620, 1, 1200, 1232], [625] * 7 + [628],
                                   [160, 320, 480, 640, 800, 960, 1120, 523], [161, 321, 481, 641, 801, 961, 1121, 516],
                                   [1500], [1100], [2304]])
@pytest.mark.parametrize("act,n,gathered", [("none", 1000, False), ("gated", 512, False), ("relu", 1096, True)])
def test_heights_of_tiles(sizes, act, n, gathered):
    """Tiles of up to 256 rows are lower where that saves a round; the groups are not what was reckoned with."""
    k, groups, used = 328, len(sizes), sum(sizes)
    both = (2,) if act == "gated" else ()
    gen = generator(used + n)
    sources = 900 if gathered else used
    a = torch.randn(sources, k, generator=gen, device="cuda").half()
    b = (torch.randn(groups, *both, n, k, generator=gen, device="cuda") * k ** -0.5).half()
    index = torch.randint(-1, sources + 1, (used,), generator=gen, device="cuda", dtype=torch.int32) if gathered else None
    offsets = torch.tensor(list(itertools.accumulate([0] + sizes)), dtype=torch.int32, device="cuda")
    base, out = kept(used, n, torch.float32)
    before = rt.form_counters()["product_256"]
    assert ec.grouped(a, offsets, b, out, act=act, index=index) == 0
    assert rt.form_counters()["product_256"] == before + (not gathered) or used < 1500   # (those of an index: 64 rows)
    av = a.double()
    if gathered:
        there = (index >= 0) & (index < sources)
        av = torch.where(there[:, None], av[index.long().clamp(0, sources - 1)], torch.zeros_like(av[:1]))
    for g in range(groups):
        lo, hi = sum(sizes[:g]), sum(sizes[:g + 1])
        if lo < hi:
            ec.close(out[lo:hi], *ec.product64(av[lo:hi], b[g].double(), None, act, torch.float32))
    assert (base[:, n:] == KEEP).all()


def test_forms_of_one_group():
    """The counters say which tiles calls take."""
    gen = generator(1)

    def one(type, m, n, k):
        before = rt.form_counters()
        if type == "e4m3":
            (a, sa), (b, sb) = ec.e4m3(gen, m, k), ec.e4m3(gen, n, k, scale=k ** -0.5, block_rows=128)
            out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
            assert ec.matmul(a, sa, b, sb, out) == 0
            ec.close(out, *ec.product64(ec.values(a, sa, 1), ec.values(b, sb, 128), None, "none", torch.bfloat16))
        else:
            a = torch.randn(m, k, generator=gen, device="cuda").to(TYPES[type])
            b = (torch.randn(1, n, k, generator=gen, device="cuda") * k ** -0.5).to(TYPES[type])
            out = torch.empty(m, n, dtype=TYPES[type], device="cuda")
            offsets = torch.tensor([0, m], dtype=torch.int32, device="cuda")
            assert ec.grouped(a, offsets, b, out) == 0
            ec.close(out, *ec.product64(a.double(), b[0].double(), None, "none", TYPES[type]))
        return [f for f, v in rt.form_counters().items() if v != before[f]]
    assert one("e4m3", 20, 4096, 2048) == ["product_32"]
    assert one("e4m3", 300, 4096, 2048) == ["product_128"]
    assert one("e4m3", 2048, 4096, 1024) == ["product_256"]
    assert one("fp16", 20, 4096, 2048) == ["product_32"]
    assert one("fp16", 600, 1000, 4096) == ["product_64"]
    assert one("fp16", 4096, 4096, 256) == ["product_256"]


# ------------------------------------------------------------------------------------------- routing
def route64(logits, k, normalise):
    l = logits.double().cpu().numpy()
    tokens, experts = l.shape
    chosen, weights = np.full((tokens, k), -1), np.zeros((tokens, k))
    rank = np.where(np.isnan(l), np.inf, l)
    pairs = [[] for _ in range(experts)]
    with np.errstate(all="ignore"):
        for t in range(tokens):
            # NaN above +inf, then values; ties to the lower expert
            at = sorted(range(experts), key=lambda e: (not np.isnan(l[t, e]), -rank[t, e], e))[:k]
            at = [e for e in at if not (l[t, e] == -np.inf)]
            if not at:
                continue
            chosen[t, :len(at)] = at
            top = l[t, at[0]]
            e = np.exp(l[t, at] - top)
            weights[t, :len(at)] = e / (e.sum() if normalise else np.exp(l[t][l[t] != -np.inf] - top).sum())
            for j, x in enumerate(at):
                pairs[x].append(t * k + j)
    offsets = np.cumsum([0] + [len(p) for p in pairs])
    flat = np.array([s for p in pairs for s in p], dtype=np.int64)
    order, position = np.full(tokens * k, -1), np.full(tokens * k, -1)
    order[:len(flat)] = flat // k
    position[flat] = np.arange(len(flat))
    return chosen, weights, offsets, order, position.reshape(tokens, k)


def check_route(logits, k, normalise, **how):
    code, chosen, weights, offsets, order, position = ec.route(logits, k, normalise, **how)
    assert code == 0
    torch.cuda.synchronize()
    c, w, o, r, p = route64(logits, k, normalise)
    assert np.array_equal(chosen.cpu().numpy(), c)
    assert np.array_equal(offsets.cpu().numpy(), o)
    assert np.array_equal(order.cpu().numpy(), r)
    assert np.array_equal(position.cpu().numpy(), p)
    got = weights.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(w))
    # exp within 2 units of the last place of an argument rounded once (as large as 200), a sum of up to 1024, a quotient
    assert np.all(np.abs(np.nan_to_num(got) - np.nan_to_num(w)) <= np.nan_to_num(w) * (200 + 40) * 2.0 ** -23 + 1e-37)


@pytest.mark.parametrize("tokens", [1, 2, 127, 128, 129, 700])
@pytest.mark.parametrize("experts,k", [(1, 1), (4, 4), (31, 3), (32, 8), (33, 2), (64, 4), (100, 7), (128, 8), (256, 8), (257, 32),
                                       (1024, 6)])
def test_route(tokens, experts, k):
    gen = generator(tokens * 1000 + experts)
    logits = torch.randn(tokens, experts, generator=gen, device="cuda") * 3
    type = list(TYPES.values())[(tokens + experts) % 3]
    logits = ec.rows_apart(logits.to(type), 1, fill=100.0)
    check_route(logits, k, tokens % 2 == 0)


def test_route_ties_masks_and_edges():
    gen = generator(5)
    for type in TYPES.values():
        logits = torch.randint(-2, 3, (300, 40), generator=gen, device="cuda").float()
        logits[logits == 0] = -0.0
        logits[7, ::2] = 0.0
        logits[0] = -math.inf                      # nothing to take
        logits[1, 3:] = -math.inf                  # fewer than k
        logits[2] = torch.finfo(type).min          # the type's lowest value is a value
        logits[3, 5:] = torch.finfo(type).min
        logits[4, 9] = math.nan
        logits[5, 9] = math.inf
        logits[6] = math.nan
        logits[8] = torch.finfo(type).max
        logits[290:] = -math.inf                   # a padded batch
        for normalise in (False, True):
            check_route(logits.to(type), 6, normalise)


def test_route_of_all_to_one_expert_and_of_nothing():
    logits = torch.zeros(3000, 16, device="cuda")
    logits[:, 11] = 5.0
    check_route(logits, 1, True)
    check_route(torch.full((300, 16), -math.inf, device="cuda"), 4, True)
    code, _, _, offsets, _, _ = ec.route(torch.empty(0, 16, device="cuda"), 4, True)
    torch.cuda.synchronize()
    assert code == 0 and (offsets == 0).all()


def test_route_of_many_tokens():
    gen = generator(6)
    logits = (torch.randn(40000, 24, generator=gen, device="cuda") * 2).bfloat16()
    check_route(logits, 3, False)


# ------------------------------------------------------------------------------------------- weighted sum
@pytest.mark.parametrize("type,out_type", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp16"), ("bf16", "fp32"),
                                           ("fp32", "fp32")])
@pytest.mark.parametrize("tokens,k,n", [(1, 1, 1), (3, 2, 64), (33, 4, 1000), (5, 32, 130), (257, 8, 2048), (70, 3, 8200)])
def test_combine(type, out_type, tokens, k, n):
    gen = generator(tokens + n)
    for aligned in (True, False):
        y_rows = max(1, tokens * k - 2)
        y = ec.rows_apart(torch.randn(y_rows, n, generator=gen, device="cuda").to(TYPES[type]), 8 if aligned else 1)
        position = torch.randint(0, y_rows, (tokens, k), generator=gen, device="cuda", dtype=torch.int32)
        position.view(-1)[::5] = -1
        position.view(-1)[3::7] = y_rows
        if tokens > 2:
            position[1] = -1
        weights = torch.rand(tokens, k, generator=gen, device="cuda")
        weights[position < 0] = math.nan           # the weight of nothing
        base, out = kept(tokens, n, TYPES[out_type], extra=8 if aligned else 3)
        assert ec.combine(y, position, weights, out) == 0
        there = (position >= 0) & (position < y_rows)
        rows = y.double()[position.long().clamp(0, y_rows - 1)]
        w = torch.where(there, weights, torch.zeros_like(weights)).double()
        want, size = (rows * w[:, :, None]).sum(1), (rows.abs() * w[:, :, None]).sum(1)
        info = torch.finfo(TYPES[out_type])
        ec.close(out, want, size * k * 2.0 ** -23 + want.abs() * info.eps / 2 * 1.001 + info.tiny)
        assert (base[:, n:].float() == torch.tensor(KEEP).to(TYPES[out_type]).float().item()).all()


# ------------------------------------------------------------------------------------------- as they are used
class Layer:
    """An expert layer in 8 bits: route, quantise the tokens in the order of their experts, gated product, quantise, second
    product, weighted sum.  Everything a call writes is allocated once."""

    def __init__(self, tokens, hidden, inner, experts, k, seed=0):
        gen = generator(seed)
        self.k, self.tokens = k, tokens
        self.w1, self.s1 = ec.e4m3(gen, experts, 2, inner, hidden, scale=hidden ** -0.5, block_rows=128)
        self.w2, self.s2 = ec.e4m3(gen, experts, hidden, inner, scale=inner ** -0.5, block_rows=128)
        self.router = torch.randn(hidden, experts, generator=gen, device="cuda") * hidden ** -0.5
        rows = tokens * k

        def eight(r, c):
            return (torch.zeros(r, -(-c // 16) * 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :c],
                    torch.full((r, ec.blocks(c)), math.nan, device="cuda"))
        self.q1, self.qs1 = eight(rows, hidden)
        self.h = torch.zeros(rows, inner, dtype=torch.bfloat16, device="cuda")
        self.q2, self.qs2 = eight(rows, inner)
        self.y = torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda")
        self.out = torch.empty(tokens, hidden, device="cuda")
        need = rt.lib().occamy_route_experts_workspace(tokens, experts, k)
        self.work = torch.empty(need, dtype=torch.uint8, device="cuda")

    def __call__(self, x, logits, stream=None):
        code, self.chosen, self.weights, self.offsets, self.order, self.position = ec.route(
            logits, self.k, True, stream, self.work)
        codes = [code,
                 ec.quantize(x, self.q1, self.qs1, index=self.order, stream=stream),
                 ec.grouped(self.q1, self.offsets, self.w1, self.h, self.qs1, self.s1, "gated", stream=stream),
                 ec.quantize(self.h, self.q2, self.qs2, stream=stream),
                 ec.grouped(self.q2, self.offsets, self.w2, self.y, self.qs2, self.s2, stream=stream),
                 ec.combine(self.y, self.position, self.weights, self.out, stream)]
        assert codes == [0] * 6
        return self.out

    def check(self, x, logits):
        """Each step against 64 bits of what the step before it left; rows of masked tokens are zeros."""
        c, w, o, order, p = route64(logits, self.k, True)
        assert np.array_equal(self.chosen.cpu().numpy(), c) and np.array_equal(self.offsets.cpu().numpy(), o)
        used = int(o[-1])
        want, s = quantize64(x[torch.from_numpy(order[:used]).cuda()], 1)
        assert np.array_equal(self.qs1[:used].double().cpu().numpy(), s)
        same_values(self.q1[:used], want)
        a1, a2 = ec.values(self.q1[:used], self.qs1[:used], 1), ec.values(self.q2[:used], self.qs2[:used], 1)
        for g in range(len(o) - 1):
            lo, hi = int(o[g]), int(o[g + 1])
            if lo < hi:
                ec.close(self.h[lo:hi], *ec.product64(a1[lo:hi], ec.values(self.w1[g], self.s1[g], 128), None, "gated",
                                                      torch.bfloat16))
                ec.close(self.y[lo:hi], *ec.product64(a2[lo:hi], ec.values(self.w2[g], self.s2[g], 128), None, "none",
                                                      torch.bfloat16))
        rows = torch.where(torch.from_numpy(p).cuda()[:, :, None] >= 0,
                           self.y.double()[torch.from_numpy(p).cuda().clamp(min=0)], 0.0)
        wd = self.weights.double()[:, :, None]
        ec.close(self.out, (rows * wd).sum(1), (rows.abs() * wd).sum(1) * (self.k + 1) * 2.0 ** -23 + 1e-37)


@pytest.mark.parametrize("tokens", [1, 5, 200, 1100])
def test_an_expert_layer(tokens):
    layer = Layer(tokens, 384, 136, 12, 3)
    gen = generator(tokens)
    x = torch.randn(tokens, 384, generator=gen, device="cuda").bfloat16()
    logits = x.float() @ layer.router
    if tokens > 4:
        logits[-tokens // 4:] = -math.inf
    layer(x, logits)
    torch.cuda.synchronize()
    layer.check(x, logits)
    if tokens > 4:
        assert (layer.out[-tokens // 4:] == 0).all()


def test_an_expert_layer_as_a_graph():
    """Captured once, replayed on other inputs; two graphs with a workspace each, at the same time."""
    layers = [Layer(150, 256, 128, 16, 2, seed) for seed in (1, 2)]
    xs = [torch.zeros(150, 256, dtype=torch.bfloat16, device="cuda") for _ in layers]
    ls = [torch.zeros(150, 16, device="cuda") for _ in layers]
    graphs, streams = [], [torch.cuda.Stream() for _ in layers]
    for layer, x, l in zip(layers, xs, ls):
        layer(x, l)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            layer(x, l)
        graphs.append(g)
    for seed in range(3):
        gen = generator(seed)
        for x, l, layer in zip(xs, ls, layers):
            x.copy_(torch.randn(150, 256, generator=gen, device="cuda"))
            l.copy_(x.float() @ layer.router)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for layer, x, l in zip(layers, xs, ls):
            layer.check(x, l)


def test_calls_on_a_stream_of_their_own():
    """Ordered by the stream they are given alone: the inputs arrive late, and the results are read behind them."""
    layer = Layer(300, 256, 128, 8, 2)
    gen = generator(8)
    x0 = torch.randn(300, 256, generator=gen, device="cuda").bfloat16()
    l0 = x0.float() @ layer.router
    x, l = torch.zeros_like(x0), torch.zeros_like(l0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        x.copy_(x0)
        l.copy_(l0)
        layer(x, l)
    s.synchronize()
    layer.check(x0, l0)


def test_the_first_call_is_not_captured():
    """In a process of its own: the call that sets the runtime up is refused while its stream is captured, and the capture goes on."""
    import os
    import subprocess
    import sys
    code = (
        "import torch, expert_calls as ec\n"
        "x = torch.randn(4, 128, device='cuda'); q = torch.zeros(4, 128, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)\n"
        "s = torch.zeros(4, 1, device='cuda'); n = torch.zeros(1, device='cuda')\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    n.add_(1)\n"
        "    first = ec.quantize(x, q, s)\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "assert first == -6 and n.item() == 1 and (s == 0).all(), (first, n.item())\n"
        "assert ec.quantize(x, q, s) == 0\n"
        "torch.cuda.synchronize(); assert (s > 0).all()\n"
        "g = torch.cuda.CUDAGraph(); s.zero_()\n"
        "with torch.cuda.graph(g):\n"
        "    assert ec.quantize(x, q, s) == 0\n"
        "g.replay(); torch.cuda.synchronize(); assert (s > 0).all()\n")
    here = os.path.dirname(os.path.abspath(__file__))
    env = {**os.environ, "PYTHONPATH": os.pathsep.join([here, os.path.dirname(here)])}
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0, r.stderr


def test_clusters_of_two_streams():
    """Calls whose tiles are shared by clusters, on two streams at a time."""
    gen = generator(21)
    calls = []
    for m, n, k in ((1, 4096, 4096), (40, 4096, 4096), (90, 2048, 8192), (3, 1000, 4096)):
        (a, sa), (b, sb) = ec.e4m3(gen, m, k), ec.e4m3(gen, n, k, scale=k ** -0.5, block_rows=128)
        out = torch.empty(m, n, device="cuda")
        assert ec.matmul(a, sa, b, sb, out) == 0
        torch.cuda.synchronize()
        ec.close(out, *ec.product64(ec.values(a, sa, 1), ec.values(b, sb, 128), None, "none", torch.float32))
        calls.append((a, sa, b, sb, out.clone(), [torch.empty_like(out) for _ in range(2)]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for a, sa, b, sb, _, outs in (calls if i else calls[::-1]):
                    assert ec.matmul(a, sa, b, sb, outs[i]) == 0
    torch.cuda.synchronize()
    for *_, want, outs in calls:
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_two_threads():
    layers = [Layer(120, 256, 128, 8, 2, seed) for seed in (3, 4)]
    gen = generator(9)
    xs = [torch.randn(120, 256, generator=gen, device="cuda").bfloat16() for _ in layers]
    ls = [x.float() @ layer.router for x, layer in zip(xs, layers)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    layers[i](xs[i], ls[i])
            s.synchronize()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for layer, x, l in zip(layers, xs, ls):
        layer.check(x, l)


def test_pointers_that_are_not_device_memory_are_refused():
    a, sa = ec.e4m3(generator(1), 16, 128)
    b, sb = ec.e4m3(generator(2), 16, 128, block_rows=128)
    out = torch.full((16, 16), KEEP, device="cuda")
    host = torch.zeros(4096)
    assert ec.matmul(a, host, b, sb, out) == -5
    assert ec.matmul(a, sa, b, sb, torch.zeros(16, 16)) == -5
    assert ec.matmul(a, sa, b, sb, out, bias=host) == -5
    torch.cuda.synchronize()
    assert (out == KEEP).all()
    odd = torch.zeros(16 * 144 + 1, dtype=torch.uint8, device="cuda")[1:].view(16, 144)[:, :128].view(torch.float8_e4m3fn)
    assert ec.matmul(odd, sa, b, sb, out) == -3


# ------------------------------------------------------------------------------------------- memory of the runtime's own
@pytest.mark.parametrize("own_stream", [True, False])
@pytest.mark.parametrize("math_mode", [rt.MATH_BF16, rt.MATH_FP32])
def test_behind_the_layers_of_a_model(own_stream, math_mode):
    """Features of a convolution and a global average pool (kept in another format by the runtime), an 8-bit classifier, its
    softmax through the ABI: without a wait in between, on the runtime's stream or another."""
    import ctypes as C
    from oracle import ref
    rt.set_math_mode(math_mode)
    L = rt.lib()
    r = np.random.Generator(np.random.PCG64(5))
    x = r.normal(size=(6, 16, 12, 12)).astype(np.float32)
    w = (r.normal(size=(256, 16, 3, 3)) * 0.12).astype(np.float32)
    bias = r.normal(size=256).astype(np.float32)
    fc = (r.normal(size=(72, 256)) * 0.06).astype(np.float32)
    bufs = {}

    def buf(name, a=None, nbytes=0):
        bufs[name] = rt.DeviceBuffer.from_numpy(a) if a is not None else rt.DeviceBuffer(nbytes)
        return bufs[name].ptr
    xd, wd, bd, fcd = buf("x", x), buf("w", w), buf("b", bias), buf("fc", fc)
    stream = L.occamy_stream() if own_stream else torch.cuda.current_stream().cuda_stream
    q, qs = buf("q", nbytes=6 * 256), buf("qs", nbytes=6 * 2 * 4)
    fq, fs = buf("fq", nbytes=72 * 256), buf("fs", nbytes=2 * 4)
    y, feat, logits, prob = (buf(n, nbytes=4 * s) for n, s in
                             (("y", 6 * 256 * 144), ("feat", 6 * 256), ("logits", 6 * 72), ("prob", 6 * 72)))
    h = C.c_void_p()
    L.cudnnCreate(C.byref(h))
    for _ in range(3):
        L.DNNConvBiasActivFunc(h, xd, rt.dims(x.shape), wd, rt.dims(w.shape), bd, rt.dims((1, 256, 1, 1)), None, 0, 1,
                               rt.dims((1, 1)), rt.dims((1, 1)), 1, y)
        L.DNNReduceFunc(h, 4, y, rt.dims((6, 256, 12, 12)), feat, rt.dims((6, 256, 1, 1)), 5)
        assert L.occamy_quantize_e4m3(fcd, rt.F32, 72, 256, 256, None, 72, 128, fq, 256, fs, stream) == 0
        assert L.occamy_quantize_e4m3(feat, rt.F32, 6, 256, 256, None, 6, 1, q, 256, qs, stream) == 0
        assert L.occamy_matmul_e4m3(q, 256, qs, fq, 256, fs, None, 6, 72, 256, 5, logits, rt.F32, 72, stream) == 0
        L.CUDASoftmaxFunc(logits, rt.dims((6, 72)), prob, rt.dims((6, 72)), 1, 2)
    got = bufs["prob"].to_numpy((6, 72))
    L.cudnnDestroy(h)
    # the classifier is exact on what it was given: bring back its own operands
    f = bufs["feat"].to_numpy((6, 256))
    want = ref.reduce_mean(ref.conv2d(x, w, bias, (1, 1), (1, 1), act=1), (6, 256, 1, 1)).reshape(6, 256)
    assert np.abs(f - want).max() <= 2e-2 * np.abs(want).max()
    q64, s64 = quantize64(torch.from_numpy(f), 1)
    w64, ws64 = quantize64(torch.from_numpy(fc), 128)
    a64 = q64 * np.repeat(s64, 128, 1)
    l64 = a64 @ (w64 * np.repeat(np.repeat(ws64, 128, 0)[:72], 128, 1)).T
    e = np.exp(l64 - l64.max(1, keepdims=True))
    # logits of a few units, off by (256 / 16 + 8) * 2^-22 of the sum of magnitudes (under 300): 2e-3 relative at most
    assert np.abs(got - e / e.sum(1, keepdims=True)).max() <= 2e-3
    assert np.abs(got.sum(1) - 1).max() < 1e-5
    for b in bufs.values():
        b.free()
    rt.set_math_mode(rt.MATH_BF16)


def test_memory_of_the_runtime_is_refused_in_a_capture():
    a, sa = ec.e4m3(generator(1), 16, 128)
    own = rt.DeviceBuffer(16 * 128 * 2)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    out = torch.zeros(4, device="cuda")
    with torch.cuda.graph(g, stream=s):
        out.add_(1)
        code = rt.lib().occamy_quantize_e4m3(own.ptr, rt.BF16, 16, 128, 128, None, 16, 1, a.data_ptr(), a.stride(0),
                                             sa.data_ptr(), s.cuda_stream)
    assert code == -6
    g.replay()
    torch.cuda.synchronize()
    own.free()
