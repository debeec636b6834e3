"""The 8-bit and grouped operators on memory that the runtime hands out: what such memory stands for may not be there yet,
and later calls of the runtime have to see what was written."""
import numpy as np
import pytest
import torch

import expert_calls as ec
from calls import Inference, rand
from helpers import max_rel_err
from occamy_b200 import runtime as rt
from oracle import ref
from test_gpu_expert_ops import quantize64, same_values

pytestmark = pytest.mark.gpu

PASSES = 10   # recorded, fused, quiet, captured once per pool block, then replayed
SHAPE = (1, 16, 12, 12)


@pytest.fixture(autouse=True)
def no_errors(native_libs):
    rt.set_math_mode(rt.MATH_F16)   # (twenty layers: bf16 storage alone would be off by 5e-2)
    rt.lib().occamy_set_cross_call_fusion(0)   # forgets what was recorded: programs that begin alike are not replayed
    rt.lib().occamy_set_cross_call_fusion(1)
    rt.last_error(clear=True)
    yield
    rt.synchronize()
    rt.set_math_mode(rt.MATH_BF16)
    assert rt.last_error(clear=True) == 0


def quantize(x, rows, cols, stream):
    """fp32 rows at address x; (q, scales) as torch tensors."""
    q = torch.zeros(rows, cols, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros(rows, ec.blocks(cols), device="cuda")
    torch.cuda.synchronize()
    assert rt.lib().occamy_quantize_e4m3(x, rt.F32, rows, cols, cols, None, rows, 1, q.data_ptr(), cols, scales.data_ptr(),
                                         stream.cuda_stream) == 0
    return q, scales


def same_quantised(got, x):
    torch.cuda.synchronize()
    want, scales = quantize64(torch.from_numpy(x), 1)
    assert np.array_equal(got[1].double().cpu().numpy(), scales)
    same_values(got[0], want)


def copy_rows(src, dst, stream):
    """A torch tensor's rows to the fp32 rows at address dst, as a weighted sum of one row each."""
    rows, cols = src.shape
    position = torch.arange(rows, dtype=torch.int32, device="cuda")
    ones = torch.ones(rows, device="cuda")
    torch.cuda.synchronize()
    assert rt.lib().occamy_combine_experts(src.data_ptr(), rt.F32, rows, cols, position.data_ptr(), ones.data_ptr(), rows, 1,
                                           cols, dst, rt.F32, cols, stream.cuda_stream) == 0
    return position, ones


class Layers:
    """Twenty convolutions of a fresh input; after layer `at` something else may happen to its result."""

    def __init__(self):
        self.w = [rand(i, 16, 16, 3, 3, scale=0.1) for i in range(20)]
        self.b = [rand(100 + i, 16) for i in range(20)]

    def run(self, x, at=None, then=None):
        with Inference() as f:
            y = f.put(x)
            for i, (w, b) in enumerate(zip(self.w, self.b)):
                y, _ = f.conv(y, SHAPE, f.put(w), w.shape, f.put(b), (1, 1), act=1)
                if i == at:
                    y = then(f, y) or y
            return f.get(y, SHAPE)

    def want(self, x, first=0):
        for w, b in zip(self.w[first:], self.b[first:]):
            x = ref.conv2d(x, w, b, (1, 1), act=1)
        return x


@pytest.mark.parametrize("at", [2, 14, 19])
def test_results_of_a_replayed_inference(at):
    """In the middle of an inference whose calls so far wait for a graph to be launched in their place, a call on another stream
    reads one of their results."""
    model, stream = Layers(), torch.cuda.Stream()
    for i in range(PASSES):
        x = rand(200 + i, *SHAPE)
        assert max_rel_err(model.run(x), model.want(x)) <= 2e-2
    seen = {}

    def then(f, y):
        seen["q"] = quantize(y, 16, 144, stream)
        seen["y"] = f.get(y, SHAPE)
    x = rand(300, *SHAPE)
    got = model.run(x, at, then)
    same_quantised(seen["q"], seen["y"].reshape(16, 144))
    assert max_rel_err(got, model.want(x)) <= 2e-2


@pytest.mark.parametrize("at", [2, 14])
def test_writes_in_a_replayed_inference(at):
    """The same, and what the call writes is the next layer's input."""
    model, stream = Layers(), torch.cuda.Stream()
    for i in range(PASSES):
        model.run(rand(200 + i, *SHAPE))
    z = rand(301, *SHAPE)
    src = torch.from_numpy(z.reshape(16, 144)).cuda()
    kept = []

    def then(f, y):
        kept.append(copy_rows(src, y, stream))
    got = model.run(rand(300, *SHAPE), at, then)
    assert max_rel_err(got, model.want(z, at + 1)) <= 2e-2


def test_operands_that_span_several_tensors():
    """Neighbours in a pool, read as the rows of one matrix: one uploaded, one a convolution's result in the runtime's own format,
    one that was never written."""
    w, b = rand(1, 16, 16, 3, 3, scale=0.1), rand(2, 16)
    stream = torch.cuda.Stream()
    for i in range(4):
        x = rand(400 + i, *SHAPE)
        with Inference() as f:
            px, pw, pb = f.put(x), f.put(w), f.put(b)
            first = f.put(x)
            assert first % 16 == 0
            y, _ = f.conv(px, SHAPE, pw, w.shape, pb, (1, 1), act=1)
            zero = f.place(x.nbytes)
            assert (y - first, zero - y) == (x.nbytes, x.nbytes)
            got = quantize(first, 48, 144, stream)
            rows = np.concatenate([x.reshape(16, 144), f.get(y, SHAPE).reshape(16, 144), np.zeros((16, 144), np.float32)])
            # the next inference finds something else where nothing is written here
            f.put(x, at=zero - f.pool.value)
        same_quantised(got, rows)


def test_results_that_span_several_tensors():
    """The same neighbours, written in one call: none of them stands for what it was before."""
    w, b = rand(1, 16, 16, 3, 3, scale=0.1), rand(2, 16)
    z = rand(3, 3, *SHAPE)
    src = torch.from_numpy(z.reshape(48, 144)).cuda()
    stream = torch.cuda.Stream()
    for i in range(4):
        x = rand(400 + i, *SHAPE)
        with Inference() as f:
            px, pw, pb = f.put(x), f.put(w), f.put(b)
            first = f.put(x)
            y, _ = f.conv(px, SHAPE, pw, w.shape, pb, (1, 1), act=1)
            zero = f.place(x.nbytes)
            kept = copy_rows(src, first, stream)
            for p, part in zip((first, y, zero), z):
                assert np.array_equal(f.get(p, SHAPE), part)
            r = f.relu(y, SHAPE)
            assert np.array_equal(f.get(r, SHAPE), np.maximum(z[1], 0))
        del kept


def test_results_over_a_tensor_that_fusion_skipped():
    """conv -> ReLU as one kernel leaves the convolution's own result unwritten; a call may write that tensor all the same."""
    x, w, b, z = rand(1, *SHAPE), rand(2, 16, 16, 3, 3, scale=0.1), rand(3, 16), rand(4, *SHAPE)
    src = torch.from_numpy(z.reshape(16, 144)).cuda()
    stream = torch.cuda.Stream()
    want = ref.conv2d(x, w, b, (1, 1), act=1)
    chains = rt.lib().occamy_fused_chains()
    for i in range(3):
        with Inference() as f:
            y, _ = f.conv(f.put(x), SHAPE, f.put(w), w.shape, f.put(b), (1, 1), act=5)
            r = f.relu(y, SHAPE)
            if i == 2:
                kept = copy_rows(src, y, stream)
                assert np.array_equal(f.get(y, SHAPE), z)
            assert max_rel_err(f.get(r, SHAPE), want) <= 2e-2
    assert rt.lib().occamy_fused_chains() > chains
    del kept


def test_a_part_of_a_tensor_that_fusion_skipped_is_not_written():
    """What the call leaves as it was is not there: reported, as a read would be."""
    x, w, b = rand(1, *SHAPE), rand(2, 16, 16, 3, 3, scale=0.1), rand(3, 16)
    src = torch.ones(15, 144, device="cuda")
    stream = torch.cuda.Stream()
    for i in range(3):
        with Inference() as f:
            y, _ = f.conv(f.put(x), SHAPE, f.put(w), w.shape, f.put(b), (1, 1), act=5)
            f.get(f.relu(y, SHAPE), SHAPE)
            if i == 2:
                kept = copy_rows(src, y, stream)
    assert rt.last_error(clear=True) == 990
    del kept


def test_captures_of_the_runtimes_stream():
    """Memory of the runtime's own is refused in a capture, of its stream too: what has to happen to it first would become part of
    the graph, and a replay could not tell the runtime what it wrote.  Other memory is captured there like anywhere."""
    x = rand(1, 16, 256)
    fresh, plain = rt.DeviceBuffer(x.nbytes), rt.DeviceBuffer.from_numpy(x)
    rt.synchronize()
    xt = torch.zeros(16, 256, device="cuda")
    q = torch.zeros(16, 256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.zeros(16, 2, device="cuda")
    own = torch.cuda.ExternalStream(rt.lib().occamy_stream())
    other = torch.cuda.Stream()

    def call(p, s, out=None):
        return rt.lib().occamy_quantize_e4m3(p, rt.F32, 16, 256, 256, None, 16, 1, out or q.data_ptr(), 256, scales.data_ptr(),
                                             s.cuda_stream)
    assert call(xt.data_ptr(), own) == 0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=own):
        codes = [call(fresh.ptr, own), call(plain.ptr, own), call(xt.data_ptr(), own, fresh.ptr), call(plain.ptr, other),
                 call(xt.data_ptr(), own)]
    assert codes == [-6, -6, -6, -6, 0]
    for i in range(3):
        x = rand(10 + i, 16, 256)
        xt.copy_(torch.from_numpy(x))
        torch.cuda.synchronize()
        g.replay()
        same_quantised((q, scales), x)
    # nothing that is put off has been done, or noted as done, meanwhile
    assert call(fresh.ptr, other) == 0
    same_quantised((q, scales), np.zeros((16, 256), np.float32))
    fresh.free()
    plain.free()


@pytest.mark.parametrize("tokens,launches", [(0, 0), (1, 1), (128, 1), (129, 2), (5000, 2)])
def test_launches_of_routing_are_counted(tokens, launches):
    logits = torch.randn(tokens, 16, device="cuda")
    before = rt.counters()["launches"]
    assert ec.route(logits, 2, True)[0] == 0
    assert rt.counters()["launches"] - before == launches
