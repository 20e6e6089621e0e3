"""``DeviceFeatureCache`` against a 64-bit restatement of the codec and a row-by-row model of the cache.  Codes, scales
and decoded bits are compared exactly (they are those of ``quantize_int8_g32`` / ``dequantize_int8_g32``)."""
import pytest
import torch

import tensorcache_b200 as tc
from tests import low_bit_plain as plain
from tests import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GROUPS = (8, 16, 24, 32, 48, 64, 128)


class Model:
    """Rows written one after the other, on the host."""

    def __init__(self, rows, width, group):
        self.group = group
        self.q = torch.zeros(rows, width, dtype=torch.float64)
        self.s = torch.zeros(rows, width // group, dtype=torch.bfloat16)

    def write(self, indices, x):
        q, s = plain.int8_encode(x.cpu(), self.group)
        for t, i in enumerate(indices.tolist()):
            if 0 <= i < self.q.shape[0]:
                self.q[i], self.s[i] = q[t], s[t]

    def read(self, indices):
        out = torch.zeros(len(indices), self.q.shape[1], dtype=torch.float64)
        v = plain.int8_values(self.q, self.s, self.group)
        for t, i in enumerate(indices.tolist()):
            if 0 <= i < self.q.shape[0]:
                out[t] = v[i]
        return out.to(torch.bfloat16)       # 15 significant bits: one rounding

    def check(self, cache):
        assert torch.equal(cache.codes.cpu().double(), self.q)
        assert torch.equal(cache.scales.cpu(), self.s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("new", [1, 37, 1500])
def test_write_and_read(group, dtype, new):
    """Both write kernels (few rows, many rows), skipped rows, repeated and out-of-range indices, rows left alone."""
    g = torch.Generator(device=DEV).manual_seed(group + new)
    rows, width = 700, group * (5 if group >= 48 else 17)
    cache, model = tc.DeviceFeatureCache(rows, width, group, DEV), Model(rows, width, group)
    for _ in range(3):
        x = (torch.randn(new, width, generator=g, device=DEV) * 3).to(dtype)
        idx = torch.randint(-3, rows + 3, (new,), generator=g, device=DEV)
        cache.write(idx, x)
        model.write(idx, x)
    model.check(cache)
    order = torch.randint(-2, rows + 2, (900,), generator=g, device=DEV)
    assert torch.equal(cache.read(order).cpu(), model.read(order))


def test_bits_are_those_of_the_codec_on_edge_values():
    x = synth.edge_values().view(8, 512).to(DEV)
    for dtype in (torch.float32, torch.bfloat16):
        cache = tc.DeviceFeatureCache(8, 512, 32, DEV)
        cache.write(torch.arange(8, device=DEV), x.to(dtype))
        q, s, shape = tc.quantize_int8_g32(x.to(dtype))
        assert torch.equal(cache.codes.view(-1), q) and torch.equal(cache.scales.view(-1).view(torch.int16), s.view(torch.int16))
        assert torch.equal(cache.read(range(8)).view(torch.int16), tc.dequantize_int8_g32(q, s, shape).view(torch.int16))


@pytest.mark.parametrize("new", [64, 5000])
def test_every_row_to_one_index(new):
    cache = tc.DeviceFeatureCache(4, 256, 32, DEV)
    x = torch.randn(new, 256, device=DEV).to(torch.bfloat16)
    for _ in range(3):
        x = x.flip(0).contiguous()
        cache.write(torch.full((new,), 2, device=DEV), x)
        q, s, _ = tc.quantize_int8_g32(x[-1])
        assert torch.equal(cache.codes[2], q) and torch.equal(cache.scales[2], s)
        assert not bool(cache.codes[[0, 1, 3]].any())


def test_samples_strides_index_types_and_buffers():
    cache = tc.DeviceFeatureCache(10, (6, 64), 32, DEV)
    x = torch.randn(3, 6, 64, device=DEV)
    cache.write([7, 0, 3], x)
    ref = cache.read([7, 0, 3])
    assert ref.shape == (3, 6, 64) and len(cache) == 10
    other = tc.DeviceFeatureCache(10, (6, 64), 32, DEV)
    wide = torch.zeros(3, 6, 131, device=DEV)
    wide[..., 1:65] = x
    other.write(torch.tensor([7, 0, 3], dtype=torch.int32), wide[..., 1:65])
    assert torch.equal(other.codes, cache.codes)
    other.write(torch.tensor([7, 9, 0, 9, 3], device=DEV, dtype=torch.int32)[::2], x.cpu().view(3, 384))
    assert torch.equal(other.codes, cache.codes)
    other.write(torch.tensor([7, 0, 3]), x.double())
    assert torch.equal(other.codes, cache.codes)
    buf = torch.full((3 * 384 + 2,), 7.0, dtype=torch.bfloat16, device=DEV)
    cache.read(torch.tensor([7, 0, 3], device=DEV), out_buffer=buf[1:-1].view(3, 6, 64))
    assert torch.equal(buf[1:-1].view(3, 6, 64), ref) and float(buf[0]) == 7 and float(buf[-1]) == 7
    host = torch.empty(3, 6, 64, dtype=torch.bfloat16)
    assert cache.read([7, 0, 3], out_buffer=host) is host and torch.equal(host, ref.cpu())
    cache.write([], torch.empty(0, 6, 64, device=DEV))
    assert cache.read([]).shape == (0, 6, 64)
    empty = tc.DeviceFeatureCache(0, 32, 32, DEV)
    assert not bool(empty.read(torch.tensor([0, -1], device=DEV)).any())
    empty.write(torch.tensor([0, 1], device=DEV), torch.ones(2, 32, device=DEV))


@pytest.mark.parametrize("new", [5, 2000])
def test_captured_write_and_read_replay_with_other_inputs(new):
    """The replays see other rows and other indices than the capture, repeated ones among them."""
    rows, width = 300, 96
    g = torch.Generator(device=DEV).manual_seed(new)
    cache, model = tc.DeviceFeatureCache(rows, width, 16, DEV), Model(rows, width, 16)
    x, idx = torch.zeros(new, width, device=DEV), torch.zeros(new, dtype=torch.int64, device=DEV)
    order = torch.arange(rows, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.write(idx, x)
        cache.read(order)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(idx, x)
        out = cache.read(order)
    cache.codes.zero_()
    cache.scales.zero_()
    for _ in range(4):
        x.copy_(torch.randn(new, width, generator=g, device=DEV))
        idx.copy_(torch.randint(-1, rows, (new,), generator=g, device=DEV))
        graph.replay()
        model.write(idx, x)
        assert torch.equal(out.cpu(), model.read(order))


def test_offsets_beyond_2_31():
    rows, width = 1_500_000, 2048          # 3.07 G codes
    cache = tc.DeviceFeatureCache(rows, width, 32, DEV)
    idx = torch.tensor([rows - 1, 0, rows - 1500, 1_048_576 + 1], device=DEV)
    x = torch.randn(4, width, device=DEV).to(torch.bfloat16)
    cache.write(idx, x)
    q, s, shape = tc.quantize_int8_g32(x)
    assert torch.equal(cache.codes[idx].view(-1), q) and torch.equal(cache.scales[idx].view(-1), s)
    assert torch.equal(cache.read(idx), tc.dequantize_int8_g32(q, s, shape))
    assert int(cache.codes.view(torch.int64).count_nonzero()) <= 4 * width // 8
    many = torch.cat([torch.full((2000,), -1, device=DEV), idx.flip(0)])
    cache.write(many, torch.cat([torch.zeros(2000, width, dtype=torch.bfloat16, device=DEV), x]))
    assert torch.equal(cache.read(idx.flip(0)), tc.dequantize_int8_g32(q, s, shape))


@pytest.mark.parametrize("new", [70, 1100])
def test_rows_that_are_whole_samples(new):
    """[446, 768] a row: several parts a row in the kernel of few rows, and more than one unit list per block in the other."""
    rows = 1200
    cache = tc.DeviceFeatureCache(rows, (446, 768), 32, DEV)
    x = torch.randn(new, 446, 768, device=DEV).to(torch.bfloat16)
    idx = torch.randperm(rows, device=DEV)[:new]
    idx[new // 2] = idx[0]                  # row 0 of x is overwritten by a later one
    cache.write(idx, x)
    out = cache.read(idx)
    assert torch.equal(out[0], out[new // 2])
    q, s, _ = tc.quantize_int8_g32(x[1:])
    assert torch.equal(out[1:], tc.dequantize_int8_g32(q, s, x[1:].shape))
    untouched = torch.ones(rows, dtype=torch.bool, device=DEV)
    untouched[idx] = False
    assert not bool(cache.codes[untouched].any()) and not bool(cache.scales[untouched].any())


def test_writes_and_reads_interleaved_on_one_stream():
    """Many calls of both write kernels and reads between them without a synchronisation: every read sees the writes ahead of it."""
    g = torch.Generator(device=DEV).manual_seed(3)
    rows, width = 3000, 64
    cache, model = tc.DeviceFeatureCache(rows, width, 16, DEV), Model(rows, width, 16)
    steps, order = [], torch.arange(rows, device=DEV)
    for i in range(24):
        new = 2500 if i % 2 else 40
        idx = torch.randint(0, rows, (new,), generator=g, device=DEV)
        steps.append((idx, torch.randn(new, width, generator=g, device=DEV)))
    torch.cuda.synchronize()
    reads = []
    for idx, x in steps:
        cache.write(idx, x)
        reads.append(cache.read(order))
    for (idx, x), out in zip(steps, reads):
        model.write(idx, x)
        assert torch.equal(out.cpu(), model.read(order))
