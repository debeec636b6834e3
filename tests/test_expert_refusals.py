"""What the 8-bit and grouped operators refuse, without a GPU: every check of arguments comes before the device."""
import ctypes as C

import pytest

from occamy_b200 import runtime as rt

P = 1 << 20   # an address that nothing reads: the calls end before


@pytest.fixture(scope="module")
def lib(native_libs):
    return rt.load_library(native_libs["runtime"])


def call(fn, good, **other):
    return fn(*{**good, **other}.values())


QUANT = dict(x=P, type=1, x_rows=8, cols=256, ldx=256, index=None, rows=8, block_rows=1, q=P, ldq=256, scales=P, stream=None)
MATMUL = dict(a=P, lda=256, scale_a=P, b=P, ldb=256, scale_b=P, bias=None, m=8, n=16, k=256, act=5, out=P, out_type=0,
              ldo=16, stream=None)
GROUPED = dict(a=P, type=1, a_rows=8, lda=256, scale_a=None, index=None, offsets=P, groups=4, b=P, ldb=256, scale_b=None,
               bias=None, rows=8, n=16, k=256, act=5, out=P, out_type=0, ldo=16, stream=None)
ROUTE = dict(logits=P, type=0, tokens=8, experts=16, ldl=16, k=2, normalise=1, chosen=P, weights=P, offsets=P, order=P,
             position=P, workspace=P, bytes=1 << 20, stream=None)
COMBINE = dict(y=P, type=1, y_rows=8, ldy=64, position=P, weights=P, tokens=4, k=2, n=64, out=P, out_type=1, ldo=64,
               stream=None)


@pytest.mark.parametrize("other", [
    dict(type=3), dict(type=-1), dict(x_rows=-1), dict(cols=-1), dict(rows=-1), dict(rows=1 << 31), dict(block_rows=0),
    dict(block_rows=64), dict(index=P, block_rows=128), dict(rows=9), dict(ldx=255), dict(ldq=255), dict(ldx=1 << 62),
    dict(x=None), dict(q=None), dict(scales=None)])
def test_quantize_refuses(lib, other):
    assert call(lib.occamy_quantize_e4m3, QUANT, **other) == -3


@pytest.mark.parametrize("other", [
    dict(m=-1), dict(n=-1), dict(k=0), dict(k=-5), dict(n=1 << 31), dict(act=4), dict(act=7), dict(act=1 << 32), dict(out_type=3),
    dict(lda=255), dict(lda=264), dict(ldb=264), dict(ldb=128), dict(ldo=15), dict(a=None), dict(b=None), dict(out=None),
    dict(scale_a=None), dict(scale_b=None), dict(lda=1 << 41), dict(ldo=1 << 60)])
def test_matmul_refuses(lib, other):
    assert call(lib.occamy_matmul_e4m3, MATMUL, **other) == -3


@pytest.mark.parametrize("other", [
    dict(type=0), dict(type=4), dict(a_rows=9), dict(index=P, a_rows=-1), dict(index=P, a_rows=0), dict(index=P, a_rows=1 << 30, lda=256), dict(rows=-1), dict(groups=-1), dict(groups=1025),
    dict(k=0), dict(act=4), dict(act=8), dict(act=7, n=20, ldo=20), dict(lda=260), dict(ldb=260), dict(out_type=3),
    dict(offsets=None), dict(a=None), dict(b=None), dict(out=None), dict(type=3), dict(type=3, scale_a=P),
    dict(groups=1024, n=1 << 22, ldo=1 << 22)])
def test_grouped_refuses(lib, other):
    assert call(lib.occamy_matmul_grouped, GROUPED, **other) == -3


@pytest.mark.parametrize("other", [
    dict(type=3), dict(tokens=-1), dict(experts=0), dict(experts=1025, ldl=1025), dict(k=0), dict(k=17),
    dict(k=33, experts=64, ldl=64), dict(ldl=15), dict(tokens=1 << 30), dict(logits=None), dict(chosen=None),
    dict(weights=None), dict(offsets=None), dict(order=None), dict(position=None)])
def test_route_refuses(lib, other):
    assert call(lib.occamy_route_experts, ROUTE, **other) == -3


def test_route_wants_its_workspace(lib):
    need = lib.occamy_route_experts_workspace(8, 16, 2)
    assert need > 0
    assert call(lib.occamy_route_experts, ROUTE, bytes=need - 1) == -2
    assert call(lib.occamy_route_experts, ROUTE, workspace=None) == -2
    assert lib.occamy_route_experts_workspace(-1, 16, 2) == -3
    assert lib.occamy_route_experts_workspace(8, 1025, 2) == -3
    assert lib.occamy_route_experts_workspace(8, 16, 33) == -3


@pytest.mark.parametrize("other", [
    dict(type=3), dict(out_type=3), dict(y_rows=-1), dict(tokens=-1), dict(n=-1), dict(k=0), dict(k=33), dict(ldy=63),
    dict(ldo=63), dict(y=None), dict(position=None), dict(weights=None), dict(out=None)])
def test_combine_refuses(lib, other):
    assert call(lib.occamy_combine_experts, COMBINE, **other) == -3


def test_empty_problems_are_done(lib):
    assert call(lib.occamy_quantize_e4m3, QUANT, rows=0, x_rows=0) == 0
    assert call(lib.occamy_quantize_e4m3, QUANT, cols=0) == 0
    assert call(lib.occamy_matmul_e4m3, MATMUL, m=0) == 0
    assert call(lib.occamy_matmul_e4m3, MATMUL, n=0) == 0
    assert call(lib.occamy_matmul_grouped, GROUPED, rows=0, a_rows=0) == 0
    assert call(lib.occamy_matmul_grouped, GROUPED, groups=0) == 0
    assert call(lib.occamy_combine_experts, COMBINE, tokens=0) == 0


@pytest.mark.parametrize("at", ["m", "n"])
def test_products_refuse_what_32_bits_do_not_number(lib, at):
    k = dict(ldo=2 ** 31) if at == "n" else {}
    assert call(lib.occamy_matmul_e4m3, MATMUL, **{at: 2 ** 31 - 1023}, **k) == -3
    grouped = dict(rows=2 ** 31 - 1023, a_rows=2 ** 31 - 1023) if at == "m" else dict(n=2 ** 31 // GROUPED["groups"], ldo=2 ** 31)
    assert call(lib.occamy_matmul_grouped, GROUPED, **grouped) == -3


def test_no_device_is_an_error(lib):
    """On a machine without a GPU the calls say so; they do not end the process."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is a GPU")
    for fn, good in ((lib.occamy_quantize_e4m3, QUANT), (lib.occamy_matmul_e4m3, MATMUL),
                     (lib.occamy_matmul_grouped, GROUPED), (lib.occamy_route_experts, ROUTE),
                     (lib.occamy_combine_experts, COMBINE)):
        assert call(fn, good) == -1


def test_header_and_binding_agree():
    """Every entry point has as many arguments here as in the header."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                             "occamy_dnn_api.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name in ("occamy_quantize_e4m3", "occamy_matmul_e4m3", "occamy_matmul_grouped", "occamy_route_experts",
                 "occamy_route_experts_workspace", "occamy_combine_experts"):
        args = re.search(name + r"\s*\(([^;]*)\)\s*;", text).group(1)
        types = rt._SIGNATURES[name][1]
        assert len(args.split(",")) == len(types), name
        for a, t in zip(args.split(","), types):
            want = C.c_void_p if "*" in a or "cudaStream_t" in a else (C.c_int64 if "int64_t" in a else C.c_int)
            assert t is want, (name, a)
