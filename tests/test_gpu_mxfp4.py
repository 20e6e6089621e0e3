"""MXFP4 codec and product against a 64-bit restatement.  Codes, scale bytes and decoded bf16 values are compared exactly: the
scale is a power of two, so the quotient and the decoded product have no rounding but the one to the E2M1 grid."""
import pytest
import torch

import tensorcache_b200 as tc
from tensorcache_b200.fused_linear import check_device_status
from tests import low_bit_plain as plain
from tests import synth
from tests.util import bits

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def check_codec(x):
    """Codes, scales, padding and decoded values of a 2-D tensor."""
    rows, cols = x.shape
    codes, scales, shape = tc.quantize_mxfp4(x)
    assert codes.shape == (rows, cols // 2) and codes.dtype == torch.uint8 and tuple(shape) == (rows, cols)
    ref_code, ref_byte = plain.mx_encode(x)
    assert torch.equal(codes, plain.mx_pack(ref_code))
    per_row = tc.mxfp4_scales_to_rows(scales, rows, cols)
    assert torch.equal(per_row.long(), ref_byte)
    assert torch.equal(tc.mxfp4_scales_from_rows(per_row), scales)      # padding is 0
    out = tc.dequantize_mxfp4(codes, scales, shape)
    assert out.dtype == torch.bfloat16 and out.shape == x.shape
    assert torch.equal(out.double(), plain.mx_values(ref_code, ref_byte))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (3, 96), (127, 128), (128, 160), (129, 992), (446, 768), (1000, 4128)])
def test_codec_matches_the_restatement(rows, cols, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g, device=DEV) * torch.exp(2 * torch.randn(rows, 1, generator=g, device=DEV))
    check_codec(x.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_grid_point_tie_and_neighbour(dtype):
    """All E2M1 values, the midpoints between them and values just beside both, in blocks whose maximum pins the scale."""
    mid = (plain.GRID[1:] + plain.GRID[:-1]) / 2
    base = torch.cat([plain.GRID, mid, torch.tensor([6.5, 7.0, 7.5], dtype=torch.float64)])
    eps = 2.0 ** (-7 if dtype == torch.bfloat16 else -10)
    v = torch.cat([base, base * (1 + eps), base * (1 - eps)])
    v = torch.cat([v, -v])
    v = v[v.abs() < 8]
    blocks = v[:v.numel() // 31 * 31].view(-1, 31)
    x = torch.cat([torch.full((blocks.shape[0], 1), 4.0, dtype=torch.float64), blocks], 1)   # max in [4, 8): scale 1
    for scale in (1.0, 2.0 ** -9, 2.0 ** 8):
        check_codec((x * scale).to(dtype).to(DEV))


def test_extremes_of_the_exponent_and_values_that_are_not_finite():
    x = synth.edge_values().view(8, 512).clone()
    x[7, :32] = torch.tensor([float("nan"), float("inf"), float("-inf"), 5.0] * 8)
    x[7, 32:64] = 3.4028e38
    x[7, 64:96] = 1.1754944e-38     # smallest normal fp32
    x[7, 96:128] = 1e-45            # smallest subnormal
    x[7, 128:160] = -0.0
    check_codec(x.to(DEV))
    check_codec(x.to(torch.bfloat16).to(DEV))
    check_codec(x.to(torch.float16).to(DEV))


def test_all_codes_and_scale_bytes_decode():
    """Every scale byte (as another program may have written them) with every code."""
    code = torch.arange(16, device=DEV).repeat(256, 2)
    byte = torch.arange(256, device=DEV).view(256, 1)
    out = tc.dequantize_mxfp4(plain.mx_pack(code), tc.mxfp4_scales_from_rows(byte.to(torch.uint8)), (256, 32))
    ref = plain.mx_values(code, byte).to(torch.bfloat16)
    assert bool(out[255].isnan().all())
    assert torch.equal(out[:255].float(), ref[:255].float())


def test_leading_dimensions_strides_alignment_buffers_and_host_tensors():
    x = synth.config0_style(3, (3, 5, 64)).to(DEV)
    codes, scales, shape = tc.quantize_mxfp4(x)
    assert codes.shape == (3, 5, 32) and tuple(shape) == (3, 5, 64)
    ref = tc.dequantize_mxfp4(codes, scales, shape)
    wide = torch.zeros(3, 5, 200, dtype=torch.bfloat16, device=DEV)
    wide[..., 7:71] = x
    for view in (wide[..., 7:71], x.transpose(0, 1).contiguous().transpose(0, 1)):
        c2, s2, _ = tc.quantize_mxfp4(view)
        assert torch.equal(c2, codes) and torch.equal(s2, scales)
    odd = torch.empty(15 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(3, 5, 64)     # 2-byte aligned
    odd.copy_(x)
    c2, s2, _ = tc.quantize_mxfp4(odd)
    assert torch.equal(c2, codes) and torch.equal(s2, scales)
    buf = torch.full((15 * 64 + 8,), 7.0, dtype=torch.bfloat16, device=DEV)
    assert tc.dequantize_mxfp4(codes, scales, shape, out_buffer=buf[1:961].view(3, 5, 64)) is not None
    assert torch.equal(buf[1:961].view(3, 5, 64), ref) and bool((buf[961:] == 7).all()) and float(buf[0]) == 7
    cc, cs, _ = tc.quantize_mxfp4(x.cpu())
    assert not cc.is_cuda and torch.equal(cc, codes.cpu()) and torch.equal(cs, scales.cpu())
    assert (bits(tc.dequantize_mxfp4(cc, cs, shape)) == bits(ref)).all()
    c64, s64, _ = tc.quantize_mxfp4(x.double())
    assert torch.equal(c64, codes) and torch.equal(s64, scales)


def test_empty_tensors():
    for shape in ((0, 64), (4, 0), (0,), (2, 0, 32)):
        codes, scales, s = tc.quantize_mxfp4(torch.empty(shape, device=DEV))
        assert codes.numel() == 0 and tc.dequantize_mxfp4(codes, scales, s).shape == shape


def test_capture_and_replay_on_another_stream():
    x = torch.randn(200, 96, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tc.dequantize_mxfp4(*tc.quantize_mxfp4(x))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tc.dequantize_mxfp4(*tc.quantize_mxfp4(x))
    for seed in (1, 2):
        x.copy_(torch.randn(200, 96, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        graph.replay()
        assert torch.equal(out.double(), plain.mx_values(*plain.mx_encode(x)))


def test_more_than_2_31_values():
    rows, cols = (1 << 20) + 3, 2080
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(131, cols, device=DEV).to(torch.bfloat16)
    x[-131:] = tail
    codes, scales, shape = tc.quantize_mxfp4(x)
    out = tc.dequantize_mxfp4(codes, scales, shape)
    assert torch.equal(out[-131:].double(), plain.mx_values(*plain.mx_encode(tail)))
    assert not bool(out[:1000].any()) and not bool(codes[:-131].any())


# ------------------------------------------------------------------------------------------------ product
#
# Tolerance: code products times powers of two are exact in fp32; adding K of them in fp32, in any order and even with
# truncation, is off by at most K 2^-23 times the sum of magnitudes; the result is rounded once to bf16 (2^-8 of it).


def product_close(got, x, w, bias=None):
    """x, w: fp64 values of the two operands."""
    ref, bound = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        ref, bound = ref + bias.double(), bound + bias.double().abs()
    tol = 2.0 ** -8 * ref.abs() + 1.01 * (x.shape[1] + 1) * 2.0 ** -23 * bound + 2.0 ** -133
    assert got.dtype == torch.bfloat16 and got.shape == ref.shape
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).nan_to_num(0).max())


def product_inputs(M, N, K, dtype=torch.bfloat16, seed=0):
    """Rows and blocks of very different sizes, so that a scale applied to the wrong row or block shows."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV) * torch.exp2(torch.randint(-4, 5, (M, K // 32, 1), generator=g, device=DEV).expand(-1, -1, 32).reshape(M, K))
    w = torch.randn(N, K, generator=g, device=DEV) * torch.exp2(torch.randint(-6, 3, (N, K // 32, 1), generator=g, device=DEV).expand(-1, -1, 32).reshape(N, K))
    return x.to(dtype), w.to(torch.bfloat16), torch.randn(N, generator=g, device=DEV).to(torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 256, 64), (1, 1000, 4096), (2, 33, 96), (7, 130, 160), (16, 512, 256), (17, 257, 288), (33, 64, 1024),
                                   (64, 4096, 512), (100, 300, 992), (128, 128, 128), (129, 255, 768), (256, 256, 256), (257, 513, 4128),
                                   (446, 1001, 768), (1000, 2000, 544)])
def test_product(M, N, K, dtype):
    x, w, b = product_inputs(M, N, K, dtype, M + N + K)
    wq, ws, _ = tc.quantize_mxfp4(w)
    X, W = plain.mx_values(*plain.mx_encode(x)), plain.mx_values(*plain.mx_encode(w))
    y = tc.mxfp4_matmul(x, wq, ws)
    check_device_status()
    product_close(y, X, W)
    product_close(tc.mxfp4_matmul(x, wq, ws, bias=b), X, W, b)


@pytest.mark.parametrize("M,N,K", [(1, 14336, 4096), (5, 4096, 14336), (16, 128, 2080), (31, 4100, 1184), (32, 700, 4096), (1, 300, 70016), (20, 130, 33024),
                                   (32, 100, 262144), (33, 100, 4096), (1, 40000, 96)])
def test_product_of_few_rows(M, N, K):
    """One part and several, parts of unequal length, sums too long for the kernel of few rows, and the sizes beside its limit."""
    x, w, b = product_inputs(M, N, K, seed=M + K)
    wq, ws, _ = tc.quantize_mxfp4(w)
    y = tc.mxfp4_matmul(x, wq, ws, bias=b)
    check_device_status()
    product_close(y, plain.mx_values(*plain.mx_encode(x)), plain.mx_values(*plain.mx_encode(w)), b)


@pytest.mark.parametrize("M,N,K", [(1, 1, 4096), (3, 127, 8192), (16, 385, 4096), (17, 250, 4096), (33, 261, 96), (97, 264, 96), (161, 272, 96),
                                   (600, 10007, 64)])
def test_product_whose_last_rows_and_columns_end_inside_a_warp(M, N, K):
    """Lanes outside the output leave the loop over the parts of a split sum, or the stores of a piece, before the others."""
    x, w, b = product_inputs(M, N, K, seed=M + N)
    wq, ws, _ = tc.quantize_mxfp4(w)
    y = tc.mxfp4_matmul(x, wq, ws, bias=b)
    check_device_status()
    product_close(y, plain.mx_values(*plain.mx_encode(x)), plain.mx_values(*plain.mx_encode(w)), b)


@pytest.mark.parametrize("M,N,K", [(1, 19300, 4096), (2, 38001, 4128), (16, 19100, 8192), (32, 19300, 2048)])
def test_product_of_few_rows_with_more_tiles_than_the_gpu_runs_at_once(M, N, K):
    """Several waves of CTAs, with the short ring that a long row of x leaves room for."""
    x, w, b = product_inputs(M, N, K, seed=N)
    wq, ws, _ = tc.quantize_mxfp4(w)
    y = tc.mxfp4_matmul(x, wq, ws, bias=b)
    check_device_status()
    product_close(y, plain.mx_values(*plain.mx_encode(x)), plain.mx_values(*plain.mx_encode(w)), b)


@pytest.mark.parametrize("M,N,K", [((1 << 20) + 3, 40, 2080), ((1 << 20) + 3, 2080, 32), (40, (1 << 20) + 3, 4128), (3, (1 << 20) + 3, 4128)])
def test_products_of_more_than_2_31_values(M, N, K):
    """More than 2^31 values of x, of the result or bytes of the weight's codes: zeros but for the last rows and columns."""
    x, w = torch.zeros(M, K, dtype=torch.bfloat16, device=DEV), torch.zeros(N, K, dtype=torch.bfloat16, device=DEV)
    xt, wt, _ = product_inputs(min(M, 130), min(N, 150), K, seed=K)
    x[-xt.shape[0]:], w[-wt.shape[0]:] = xt, wt
    wq, ws, _ = tc.quantize_mxfp4(w)
    y = tc.mxfp4_matmul(x, wq, ws)
    check_device_status()
    product_close(y[-xt.shape[0]:, -wt.shape[0]:], plain.mx_values(*plain.mx_encode(xt)), plain.mx_values(*plain.mx_encode(wt)))
    if M > 130:
        assert not bool(y[:1000].any())
    if N > 150:
        assert not bool(y[:, :1000].any())


def test_scales_that_pad_a_row_do_not_reach_the_sums():
    """K = 32 in a tile of 128: the other three scales of a row are padding."""
    for M in (3, 40):
        x, w, _ = product_inputs(M, 50, 32, seed=M)
        wq, ws, _ = tc.quantize_mxfp4(w)
        rows = torch.full((128, 4), 254, dtype=torch.uint8, device=DEV)      # the largest finite scale wherever nothing is stored
        rows[:50, :1] = tc.mxfp4_scales_to_rows(ws, 50, 32)
        loud = tc.mxfp4_scales_from_rows(rows)
        assert torch.equal(tc.mxfp4_matmul(x, wq, loud), tc.mxfp4_matmul(x, wq, ws))


def test_product_of_the_identity_returns_the_weight():
    """One non-zero code per row of x, with its own scale: every weight and every scale comes back where it belongs."""
    K, N = 1024, 700
    _, w, _ = product_inputs(1, N, K, seed=3)
    wq, ws, shape = tc.quantize_mxfp4(w)
    scale = torch.exp2(torch.arange(K, device=DEV) % 13 - 6)
    y = tc.mxfp4_matmul(torch.diag(scale).to(torch.bfloat16), wq, ws)
    assert torch.equal(y.double(), (tc.dequantize_mxfp4(wq, ws, shape).double() * scale).t())


def test_product_with_many_tiles_per_pair():
    M, N, K = 5000, 6000, 640
    x, w, _ = product_inputs(M, N, K, seed=4)
    wq, ws, _ = tc.quantize_mxfp4(w)
    y = tc.mxfp4_matmul(x, wq, ws)
    check_device_status()
    product_close(y, plain.mx_values(*plain.mx_encode(x)), plain.mx_values(*plain.mx_encode(w)))


def test_product_leading_dimensions_strides_empty_and_zero_rows():
    x, w, b = product_inputs(12, 40, 96, seed=5)
    wq, ws, _ = tc.quantize_mxfp4(w)
    ref = tc.mxfp4_matmul(x, wq, ws, b)
    assert torch.equal(tc.mxfp4_matmul(x.view(2, 3, 2, 96), wq, ws, b), ref.view(2, 3, 2, 40))
    assert torch.equal(tc.mxfp4_matmul(x.t().contiguous().t(), wq, ws, b), ref)
    assert tc.mxfp4_matmul(x[0], wq, ws, b).shape == (40,) and torch.equal(tc.mxfp4_matmul(x[0], wq, ws, b), ref[0])
    shifted = torch.empty(12 * 96 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(12, 96)
    shifted.copy_(x)
    odd = [torch.empty(t.numel() + 3, dtype=torch.uint8, device=DEV)[3:] for t in (wq, ws)]
    odd[0].copy_(wq.view(-1)), odd[1].copy_(ws)
    assert torch.equal(tc.mxfp4_matmul(shifted, odd[0].view_as(wq), odd[1], b), ref)
    assert tc.mxfp4_matmul(x[:0], wq, ws, b).shape == (0, 40)
    assert tc.mxfp4_matmul(x, wq[:0], ws[:0]).shape == (12, 0)
    x[3] = 0
    x[4, 5] = float("nan")
    x[5, 6] = float("inf")
    y = tc.mxfp4_matmul(x, wq, ws)
    assert not bool(y[3].any()) and bool(y.isfinite().all())
    product_close(y, plain.mx_values(*plain.mx_encode(x)), plain.mx_values(*plain.mx_encode(w)))


def test_product_captured_and_replayed():
    x, w, b = product_inputs(40, 300, 512, seed=6)
    wq, ws, _ = tc.quantize_mxfp4(w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tc.mxfp4_matmul(x, wq, ws, b)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(tc.mxfp4_matmul(x, wq, ws, b))
    for seed in (7, 8):
        x.copy_(product_inputs(40, 300, 512, seed=seed)[0])
        want = tc.mxfp4_matmul(x, wq, ws, b)
        for graph in graphs:
            graph.replay()
        assert all(torch.equal(o, want) for o in outs)


def test_product_refusals_on_the_gpu():
    x, w, b = product_inputs(4, 8, 64)
    wq, ws, _ = tc.quantize_mxfp4(w)
    with pytest.raises(ValueError, match="no gradient"):
        tc.mxfp4_matmul(x.clone().requires_grad_(True), wq, ws)
    with torch.no_grad():
        tc.mxfp4_matmul(x.clone().requires_grad_(True), wq, ws)
    with pytest.raises(ValueError, match="x is on"):
        tc.mxfp4_matmul(x.cpu(), wq, ws)
    with pytest.raises(ValueError, match="bias"):
        tc.mxfp4_matmul(x, wq, ws, b.cpu())


def test_features_through_4_and_8_bits_together():
    """The operators as a program strings them: rows into the device cache, gathered, a head trained on their codes, the
    trained head stored in 4 bits and applied to the decoded rows."""
    cache = tc.DeviceFeatureCache(256, 64, 32, DEV)
    cache.write(torch.arange(256, device=DEV), torch.randn(256, 64, device=DEV))
    pick = torch.randperm(256, device=DEV)[:100]
    w = torch.randn(16, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    y = tc.fused_dequant_linear(cache.codes[pick], cache.scales[pick], w)
    (dw,) = torch.autograd.grad(y, [w], y.detach())
    trained = (w - 0.01 * dw).detach()
    wq, ws, _ = tc.quantize_mxfp4(trained)
    rows = cache.read(pick)
    product_close(tc.mxfp4_matmul(rows, wq, ws), plain.mx_values(*plain.mx_encode(rows)), plain.mx_values(*plain.mx_encode(trained)))


def test_trainable_operands_without_a_gradient_are_refused_in_grad_mode_only():
    x, w, b = product_inputs(4, 8, 64)
    wq, ws, _ = tc.quantize_mxfp4(w)
    want = tc.mxfp4_matmul(x, wq, ws, b)
    bias = torch.nn.Parameter(b)
    with pytest.raises(ValueError, match="bias has no gradient"):
        tc.mxfp4_matmul(x, wq, ws, bias)
    with torch.no_grad():
        assert torch.equal(tc.mxfp4_matmul(x, wq, ws, bias), want)
    assert torch.equal(tc.mxfp4_matmul(x, wq, ws, bias.detach()), want)
    q, s, _ = tc.quantize_int8_g32(x)
    s.requires_grad_(True)
    with pytest.raises(ValueError, match="scales has no gradient"):
        tc.fused_dequant_linear(q.view(4, 64), s, w)
    with torch.no_grad():
        assert torch.equal(tc.fused_dequant_linear(q.view(4, 64), s, w), tc.fused_dequant_linear(q.view(4, 64), s.detach(), w))
    weight = torch.randn(8, 64, device=DEV).to(torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(weight, torch.ones_like(weight))
        for call in (lambda: tc.fused_dequant_linear(q.view(4, 64), s.detach(), dual), lambda: tc.int8_checkpoint_linear(weight, dual),
                     lambda: tc.int8_checkpoint_linear(dual, weight)):
            with pytest.raises((NotImplementedError, RuntimeError)):
                call()
