"""Linear layers whose input is kept in 8 bits, against 64-bit products.

Tolerances.  A result is rounded once to bf16: 2^-8 of its magnitude.  The sums behind it are fp32 over bf16 x bf16
products (exact in fp32): adding n terms in fp32 in any order is off by at most n 2^-24 times the sum of magnitudes.
The weight gradient multiplies the codec's decoded values, which are bf16 roundings of code * scale: the reference
rounds them too.  With bound = |a| @ |b| that gives, per element,
    |got - ref| <= 2^-8 |ref| + (1 + 2^-8) n 2^-24 bound + smallest bf16 subnormal."""
import pytest
import torch

import tensorcache_b200 as tc
from tensorcache_b200.fused_linear import check_device_status
from tests import low_bit_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def close(got, a, b, add=None):
    """got ~ a @ b (+ add) for fp64 a [r, n], b [n, c]."""
    ref, bound = a @ b, a.abs() @ b.abs()
    if add is not None:
        ref, bound = ref + add, bound + add.abs()
    n = a.shape[1] + 1
    tol = 2.0 ** -8 * ref.abs() + 1.01 * n * 2.0 ** -24 * bound + 2.0 ** -133
    assert got.dtype == torch.bfloat16 and got.shape == ref.shape
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), (float((off / tol).nan_to_num(0).max()), tuple(got.shape))


def layer(M, N, K, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV) * torch.exp(torch.randn(K, generator=g, device=DEV))
    w = torch.randn(N, K, generator=g, device=DEV) * K ** -0.5
    return (x.to(torch.bfloat16), w.to(torch.bfloat16), torch.randn(N, generator=g, device=DEV).to(torch.bfloat16),
            torch.randn(M, N, generator=g, device=DEV).to(torch.bfloat16))


def decoded(q, s, G, zp=None):
    return plain.int8_values(q, s, G, zp).to(torch.bfloat16).double()


SIZES = [(1, 1, 16, 16), (1, 768, 768, 32), (3, 17, 96, 32), (64, 64, 64, 64), (65, 130, 80, 16), (129, 257, 384, 128), (256, 256, 256, 32),
         (257, 1000, 768, 32), (446, 768, 768, 16), (1000, 33, 2048, 64), (4000, 40, 128, 128), (20011, 100, 192, 32), (300, 2049, 1024, 32)]


@pytest.mark.parametrize("M,N,K,G", SIZES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_checkpoint_linear(M, N, K, G, with_bias):
    x, w, b, dy = layer(M, N, K, M + N + K)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = tc.int8_checkpoint_linear(x, w, b if with_bias else None, group_size=G)
    grads = torch.autograd.grad(y, [x, w] + ([b] if with_bias else []), dy)
    check_device_status()
    X, W, D = x.detach().double(), w.detach().double(), dy.double()
    close(y.detach(), X, W.t(), b.detach().double() if with_bias else None)
    close(grads[0], D, W)
    close(grads[1], D.t(), decoded(*plain.int8_encode(x.detach(), G), G))
    if with_bias:
        close(grads[2].view(1, -1), torch.ones(1, M, dtype=torch.float64, device=DEV), D)


@pytest.mark.parametrize("M,N,K,G", SIZES)
@pytest.mark.parametrize("zp", [False, True])
def test_gradient_from_cached_codes(M, N, K, G, zp):
    x, w, b, dy = layer(M, N, K, M + N)
    w.requires_grad_(True), b.requires_grad_(True)
    if zp:
        q, s, z, _ = tc.compress(x, "fast", G)
    else:
        (q, s, _), z = tc.quantize_int8_g32(x, G), None
    q = q.view(M, K)
    y = tc.fused_dequant_linear(q, s, w, b, zero_points=z, group_size=G)
    dw, db = torch.autograd.grad(y, [w, b], dy)
    check_device_status()
    X = decoded(q, s, G, z)
    close(y.detach(), X, w.detach().double().t(), b.detach().double())
    close(dw, dy.double().t(), X)
    close(db.view(1, -1), torch.ones(1, M, dtype=torch.float64, device=DEV), dy.double())
    # the values of the module without gradients
    module = tc.FusedDequantLinear(K, N, group_size=G).to(DEV)
    with torch.no_grad():
        module.weight.copy_(w), module.bias.copy_(b)
    assert torch.equal(module(q, s, z), y.detach())


def test_wide_layer():
    """Many tiles per pair of CTAs (both accumulators, several bands of tiles) in all three products."""
    M, N, K, G = 4360, 2312, 2560, 32
    x, w, _, dy = layer(M, N, K)
    x.requires_grad_(True), w.requires_grad_(True)
    y = tc.int8_checkpoint_linear(x, w, None, group_size=G)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    X, W, D = x.detach().double(), w.detach().double(), dy.double()
    close(y.detach(), X, W.t())
    close(dx, D, W)
    close(dw, D.t(), decoded(*plain.int8_encode(x.detach(), G), G))


def test_gradients_against_differences():
    """Directional differences of the layer's own outputs.  The loss is linear in w and in x, so a difference over a
    finite step is exact but for the bf16 roundings of the two outputs: half a step, 2^-8 of each at most per element,
    times |dy|, summed over all elements, and of the gradient (2^-8 of each term)."""
    M, N, K = 96, 48, 64
    x, w, b, dy = layer(M, N, K, 5)
    x = (x.float() / x.float().abs().amax(-1, keepdim=True).clamp(min=1e-3) * 127).round().to(torch.bfloat16)   # codes of scale 1: exact
    x[:, ::32] = 127.0
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = tc.int8_checkpoint_linear(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], dy)
    for grad, which in ((gx, 0), (gw, 1), (gb, 2)):
        args = [x.detach(), w.detach(), b.detach()]
        step = torch.randn_like(args[which].float()).to(torch.bfloat16)
        moved = (args[which].double() + step.double()).to(torch.bfloat16)
        real = moved.double() - args[which].double()          # the step that was taken after rounding
        args[which] = moved
        y2 = tc.int8_checkpoint_linear(*args)
        change = ((y2.double() - y.detach().double()) * dy.double()).sum()
        slope = (grad.double() * real).sum()
        tol = (2.0 ** -8 * (y2.double().abs() + y.detach().double().abs()) * dy.double().abs()).sum() + (2.0 ** -8 * (grad.double() * real).abs()).sum()
        assert abs(float(change - slope)) <= float(tol)


def test_graph_keeps_codes_and_not_the_input():
    x, w, _, _ = layer(4096, 64, 1024)
    w.requires_grad_(True)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        tc.int8_checkpoint_linear(x, w)
    assert sum(t.numel() * t.element_size() for t in kept) == 4096 * 1024 * (1 + 2 / 32)
    kept.clear()
    with torch.no_grad(), torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        tc.int8_checkpoint_linear(x, w)
    assert not kept


def test_shapes_strides_partial_gradients_and_expanded_dy():
    x, w, b, dy = layer(24, 40, 64, 9)
    ref = tc.int8_checkpoint_linear(x, w, b)
    x3 = x.view(2, 3, 4, 64)
    assert torch.equal(tc.int8_checkpoint_linear(x3, w, b), ref.view(2, 3, 4, 40))
    assert torch.equal(tc.int8_checkpoint_linear(x.t().contiguous().t(), w.t().contiguous().t(), b), ref)
    shifted = torch.empty(24 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(24, 64)
    shifted.copy_(x)
    assert torch.equal(tc.int8_checkpoint_linear(shifted, w, b), ref)
    assert tc.int8_checkpoint_linear(x[0], w, b).shape == (40,)
    for which in range(3):       # one leaf at a time, a dy without memory of its own
        leaves = [x.clone(), w.clone(), b.clone()]
        leaves[which].requires_grad_(True)
        tc.int8_checkpoint_linear(*leaves).sum().backward()
        ones = torch.ones(24, 40, dtype=torch.float64, device=DEV)
        if which == 0:
            close(leaves[0].grad, ones, w.double())
        elif which == 1:
            close(leaves[1].grad, ones.t(), decoded(*plain.int8_encode(x, 32), 32))
        else:
            assert torch.equal(leaves[2].grad, torch.full_like(b, 24))
    x.requires_grad_(True), w.requires_grad_(True)
    dyt = dy.t().contiguous().t()
    a = torch.autograd.grad(tc.int8_checkpoint_linear(x, w), [x, w], dy)
    c = torch.autograd.grad(tc.int8_checkpoint_linear(x, w), [x, w], dyt)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("M,N", [(1, 1), (17, 130), (5000, 100), (40000, 9), (3001, 700)])
def test_bias_gradient_alone_and_beside_the_weight_gradient(M, N):
    x, w, b, dy = layer(M, N, 64, M)
    b.requires_grad_(True)
    (alone,) = torch.autograd.grad(tc.int8_checkpoint_linear(x, w, b), [b], dy)
    w.requires_grad_(True)
    _, beside = torch.autograd.grad(tc.int8_checkpoint_linear(x, w, b), [w, b], dy)
    for got in (alone, beside):
        close(got.view(1, -1), torch.ones(1, M, dtype=torch.float64, device=DEV), dy.double())


@pytest.mark.parametrize("M,N", [(130, 13), (4097, 101)])
def test_padding_between_rows_of_dy_is_never_used(M, N):
    """Rows of an odd number of gradients are copied to rows of a multiple of eight; the memory in between may hold NaN."""
    x, w, b, dy = layer(M, N, 64, M)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = tc.int8_checkpoint_linear(x, w, b)
    torch.cuda.synchronize()
    for size in (M * 16, M * 104, M * 64, 64 * N, 1 << 20, 1 << 22):      # what the pass is about to take from the allocator's cache
        torch.full((size,), float("nan"), dtype=torch.bfloat16, device=DEV)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], dy)
    close(gx, dy.double(), w.detach().double())
    close(gw, dy.double().t(), decoded(*plain.int8_encode(x.detach(), 32), 32))
    close(gb.view(1, -1), torch.ones(1, M, dtype=torch.float64, device=DEV), dy.double())


def test_empty_batches_and_layers():
    w, b = (torch.randn(s, device=DEV).to(torch.bfloat16).requires_grad_(True) for s in ((8, 32), (8,)))
    x = torch.empty(0, 32, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = tc.int8_checkpoint_linear(x, w, b)
    assert y.shape == (0, 8)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert gx.shape == (0, 32) and not bool(gw.any()) and not bool(gb.any()) and gw.shape == (8, 32)
    x = torch.randn(4, 32, device=DEV).to(torch.bfloat16).requires_grad_(True)
    w0 = torch.empty(0, 32, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = tc.int8_checkpoint_linear(x, w0)
    gx, gw = torch.autograd.grad(y, [x, w0], torch.empty_like(y))
    assert y.shape == (4, 0) and not bool(gx.any()) and gw.shape == (0, 32)
    q, s, _ = tc.quantize_int8_g32(x[:0])
    y = tc.fused_dequant_linear(q.view(0, 32), s, w, b)
    gw, gb = torch.autograd.grad(y, [w, b], torch.empty_like(y))
    assert not bool(gw.any()) and not bool(gb.any())


def test_repeated_calls_give_the_same_bits():
    x, w, b, dy = layer(20011, 100, 192, 1)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    runs = [torch.autograd.grad(tc.int8_checkpoint_linear(x, w, b), [x, w, b], dy) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], other))


def test_training_step_captured_and_replayed():
    M, N, K = 3000, 72, 128
    x, w, b, dy = layer(M, N, K, 3)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)

    def step():
        y = tc.int8_checkpoint_linear(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, [x, w, b], dy))

    # no eager graph of the same leaves is alive here: torch ties a leaf's gradient node to the stream of the first graph
    # that is still alive, and refuses a capture that would have to wait for that stream (for its own operators as well)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12):
        nx, nw, nb, ndy = layer(M, N, K, seed)
        with torch.no_grad():
            x.copy_(nx), w.copy_(nw), b.copy_(nb), dy.copy_(ndy)
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(out, step()))


def test_weight_changed_in_place_before_the_backward_pass_is_reported():
    x, w, _, dy = layer(16, 8, 32)
    x.requires_grad_(True)
    y = tc.int8_checkpoint_linear(x, w)
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], dy)


def test_calls_from_threads_that_have_made_no_cuda_call():
    """A fresh host thread has no CUDA context of its own until a call binds one (the memory comes from a cache)."""
    import threading

    x, w, b, dy = layer(64, 32, 64)
    q, s, _ = tc.quantize_int8_g32(x)
    calls = [lambda: tc.int8_checkpoint_linear(x, w, b), lambda: tc.fused_dequant_linear(q.view(64, 64), s, w, b),
             lambda: tc.fused_dequant_matmul(x, q.view(64, 64), s)]
    want = [c() for c in calls]
    got, errors = [None] * len(calls), []

    def work(i):
        try:
            got[i] = calls[i]()
        except Exception as e:  # noqa: BLE001 -- reported below
            errors.append(e)

    for i in range(len(calls)):
        t = threading.Thread(target=work, args=(i,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert not errors and all(torch.equal(a, c) for a, c in zip(want, got))


def test_step_on_another_stream():
    """Forward and backward on a side stream, with work of the default stream ahead of it and behind it."""
    x, w, b, dy = layer(700, 136, 256, 4)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    want = torch.autograd.grad(tc.int8_checkpoint_linear(x, w, b), [x, w, b], dy)
    side = torch.cuda.Stream()
    for _ in range(3):
        big = torch.randn(4096, 4096, device=DEV) @ torch.randn(4096, 4096, device=DEV)     # the side stream runs beside this
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = torch.autograd.grad(tc.int8_checkpoint_linear(x, w, b), [x, w, b], dy)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, c) for a, c in zip(want, got)) and big.shape == (4096, 4096)


def test_capture_with_forks_joins_copies_and_fills_between_the_kernels():
    """Kernels that may start under their predecessor, captured where that predecessor is a copy, a fill or a join of two
    streams."""
    x, w, b, dy = layer(300, 64, 128, 6)
    wq, ws, _ = tc.quantize_mxfp4(w)
    base, kept = x.clone(), torch.empty_like(x)

    def run(side):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            doubled = x * 2
            other = tc.mxfp4_matmul(doubled, wq, ws, b)
        kept.zero_()
        a = tc.int8_checkpoint_linear(x, w, b)
        main.wait_stream(side)
        c = tc.mxfp4_matmul(doubled, wq, ws, b)
        kept.copy_(doubled)
        d = tc.int8_checkpoint_linear(kept, w)
        kept.fill_(1)
        e = tc.dequantize_mxfp4(*tc.quantize_mxfp4(kept))
        return other, a, c, d, e

    side = torch.cuda.Stream()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        run(side)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(side)
    for scale in (1.0, 0.5, -2.0):
        x.copy_(base * scale)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(g, e) for g, e in zip(got, run(side)))


def test_values_that_are_not_finite_reach_the_output_but_not_the_weight_gradient():
    x, w, _, dy = layer(40, 24, 64, 8)
    x[3, 5], x[4, 6] = float("inf"), float("nan")
    w.requires_grad_(True)
    y = tc.int8_checkpoint_linear(x, w)
    (dw,) = torch.autograd.grad(y, [w], dy)
    bad = ~y.detach().isfinite().all(1)
    assert bad.nonzero().flatten().tolist() == [3, 4]
    close(dw, dy.double().t(), decoded(*plain.int8_encode(x, 32), 32))


def test_gradients_of_gradients_are_refused():
    x, w, _, _ = layer(8, 8, 32)
    x.requires_grad_(True), w.requires_grad_(True)
    (gx,) = torch.autograd.grad(tc.int8_checkpoint_linear(x, w).float().square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        gx.float().sum().backward()
    q, s, _ = tc.quantize_int8_g32(x.detach())
    (gw,) = torch.autograd.grad(tc.fused_dequant_linear(q.view(8, 32), s, w).float().square().sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError):
        gw.float().sum().backward()


def test_cached_codes_with_leading_dimensions():
    x, w, b, dy = layer(24, 40, 64, 2)
    w.requires_grad_(True), b.requires_grad_(True)
    q, s, z, _ = tc.compress(x, "fast", 32)
    want = tc.fused_dequant_linear(q.view(24, 64), s, w, b, zero_points=z)
    got = tc.fused_dequant_linear(q.view(2, 3, 4, 64), s.view(2, 3, 4, 2), w, b, zero_points=z.view(2, 3, 4, 2))
    assert torch.equal(got, want.view(2, 3, 4, 40))
    a, c = torch.autograd.grad(want, [w, b], dy), torch.autograd.grad(got, [w, b], dy.view(2, 3, 4, 40))
    assert all(torch.equal(u, v) for u, v in zip(a, c))


def test_module_trains_in_a_stack():
    """Input gradient through two layers and a non-linearity between them, against the same stack in 64 bits on the
    bf16 intermediates (so that each product is checked on its own)."""
    torch.manual_seed(0)
    l1, l2 = tc.Int8CheckpointLinear(64, 96).to(DEV), tc.Int8CheckpointLinear(96, 8, bias=False).to(DEV)
    x = torch.randn(50, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    h = l1(x)
    h.retain_grad()
    a = torch.relu(h)
    y = l2(a)
    dy = torch.randn_like(y)
    y.backward(dy)
    close(l2.weight.grad, dy.double().t(), decoded(*plain.int8_encode(a.detach(), 32), 32))
    close(l1.weight.grad, h.grad.double().t(), decoded(*plain.int8_encode(x.detach(), 32), 32))
    close(x.grad, h.grad.double(), l1.weight.detach().double())
    close(l1.bias.grad.view(1, -1), torch.ones(1, 50, dtype=torch.float64, device=DEV), h.grad.double())


def test_device_cache_feeds_a_head():
    """Rows written into a device cache, gathered as codes, and a head trained on them: the gradient is that of the
    decoded rows."""
    cache = tc.DeviceFeatureCache(500, 128, 32, DEV)
    cache.write(torch.randperm(500, device=DEV), torch.randn(500, 128, device=DEV))
    pick = torch.randint(0, 500, (77,), device=DEV)
    w = torch.randn(10, 128, device=DEV).to(torch.bfloat16).requires_grad_(True)
    dy = torch.randn(77, 10, device=DEV).to(torch.bfloat16)
    y = tc.fused_dequant_linear(cache.codes[pick], cache.scales[pick], w)
    (dw,) = torch.autograd.grad(y, [w], dy)
    rows = cache.read(pick).double()
    close(y.detach(), rows, w.detach().double().t())
    close(dw, dy.double().t(), rows)


@pytest.mark.parametrize("M", [1, 31, 33, 97, 161, 255])
@pytest.mark.parametrize("N", [261, 264, 272])
def test_last_rows_that_end_inside_a_warp(M, N):
    """Lanes whose rows lie outside the output skip the stores of a piece (staged, 16-byte and 32-byte ones); the warp has
    more pieces to read from tensor memory after it, in every product and in the parts of a split sum."""
    K = 512 + 16
    x, w, b, dy = layer(M, N, K, M + N)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = tc.int8_checkpoint_linear(x, w, b, group_size=16)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    q, s = plain.int8_encode(x.detach(), 16)
    fused = tc.fused_dequant_linear(q.to(torch.int8), s, w, b, group_size=16)
    as_weight = tc.fused_dequant_matmul(w.detach(), q.to(torch.int8), s, group_size=16)
    check_device_status()
    X, W, D, Q = x.detach().double(), w.detach().double(), dy.double(), decoded(q, s, 16)
    close(y.detach(), X, W.t(), b.detach().double())
    close(dx, D, W)
    close(dw, D.t(), Q)
    close(fused.detach(), Q, W.t(), b.detach().double())
    close(as_weight, W, Q.t())


LOWEST = torch.finfo(torch.bfloat16).min


@pytest.mark.parametrize("M,N,K,G", [(70, 24, 96, 16), (300, 260, 512, 32), (513, 40, 256, 128)])
def test_rows_of_the_lowest_value_that_no_gradient_reaches(M, N, K, G):
    """Padding of the type's lowest value (and of its neighbours) is finite: with dy = 0 it adds nothing to a gradient."""
    x, w, _, dy = layer(M, N, K, M)
    out = torch.zeros(M, dtype=torch.bool, device=DEV)
    out[::7] = out[-3:] = True
    x[out] = LOWEST
    x[0], x[7] = 3.0e38, -1.0e37
    x[14, : K // 2], x[14, K // 2 :] = LOWEST, 0.0
    dy[out] = 0
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(tc.int8_checkpoint_linear(x, w, group_size=G), [w], dy)
    check_device_status()
    close(dw, dy[~out].double().t(), decoded(*plain.int8_encode(x[~out], G), G))
    q, s, _ = tc.quantize_int8_g32(x, G)
    (dw2,) = torch.autograd.grad(tc.fused_dequant_linear(q.view(M, K), s, w, group_size=G), [w], dy)
    assert torch.equal(dw2, dw)


@pytest.mark.parametrize("zp", [False, True])
@pytest.mark.parametrize("G", [16, 32, 64, 128])
def test_groups_of_very_large_values_decode_as_elsewhere(G, zp):
    """Scales up to 2^121: every code of the group keeps the value that the decoding functions give it, zeros among them,
    in the forward product and in the weight gradient, and in the product with a quantised weight."""
    M, N, K = 66, 40, 256
    x, w, _, dy = layer(M, N, K, G)
    w, dy = (w * 2.0 ** -20).requires_grad_(True), dy * 2.0 ** -20
    big = torch.tensor([1e30, 1e34, 2e36, 1e37, 1e38, 3e38], device=DEV)
    x = torch.rand(M, K, device=DEV) * 2 - 1
    x = x * big[torch.randint(0, 6, (M, K // G, 1), device=DEV)].expand(-1, -1, G).reshape(M, K)
    x[:, 1::3] = 0.0
    x[:, ::G] = x[:, ::G].abs()
    x = x.to(torch.bfloat16)
    if zp:
        q, s, z, shape = tc.compress(x.float().clamp(min=-1e38, max=1e38).to(torch.bfloat16), "fast", G)
        X = tc.decompress(q, s, shape, z, G).double()
    else:
        (q, s, shape), z = tc.quantize_int8_g32(x, G), None
        X = tc.dequantize_int8_g32(q, s, shape, G).double()
    assert bool(X.isfinite().all()) and float(s.float().max()) > 2.0 ** 113      # beyond this, 2^15 scales are more than fp32 holds
    y = tc.fused_dequant_linear(q.view(M, K), s, w, zero_points=z, group_size=G)
    (dw,) = torch.autograd.grad(y, [w], dy)
    check_device_status()
    close(y.detach(), X, w.detach().double().t())
    close(dw, dy.double().t(), X)
    close(tc.fused_dequant_matmul(w.detach(), q.view(M, K), s, z, group_size=G), w.detach().double(), X.t())


def test_values_past_the_largest_number_stay_at_it_and_infinite_scales_are_not_hidden():
    """127 times a scale of 2.68e36 is finite in fp32 and not in bf16."""
    x = torch.full((4, 32), LOWEST, dtype=torch.bfloat16, device=DEV)
    q, s, _ = tc.quantize_int8_g32(x)
    w = torch.full((8, 32), 2.0 ** -10, dtype=torch.bfloat16, device=DEV)
    close(tc.fused_dequant_linear(q.view(4, 32), s, w), torch.full((4, 32), LOWEST, dtype=torch.float64, device=DEV), w.double().t())
    s[1], s[2] = float("inf"), float("nan")
    y = tc.fused_dequant_linear(q.view(4, 32), s, w)
    assert y.isfinite().all(1).tolist() == [True, False, False, True]


@pytest.mark.parametrize("new", [3, 1500])
def test_cache_written_before_the_backward_pass_is_reported(new):
    """The kernels write through raw addresses; the graph of a layer on the cache's own codes has to notice."""
    cache = tc.DeviceFeatureCache(2000, 64, 32, DEV)
    rows = torch.arange(new, device=DEV)
    x = torch.randn(new, 64, device=DEV)
    cache.write(rows, x)
    w = torch.randn(8, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    y = tc.fused_dequant_linear(cache.codes, cache.scales, w)
    picked = tc.fused_dequant_linear(cache.codes[rows], cache.scales[rows], w)       # copies: later writes do not matter
    cache.read(rows)
    torch.autograd.grad(y, [w], torch.ones_like(y), retain_graph=True)               # a read is not a change
    cache.write(rows, x + 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [w], torch.ones_like(y))
    torch.autograd.grad(picked, [w], torch.ones_like(picked))
    scales = cache.scales.view(-1)
    y = tc.fused_dequant_linear(cache.codes.clone(), scales, w)                      # a view of the scales alone
    cache.write(rows, x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [w], torch.ones_like(y))
    with torch.inference_mode():                                                     # tensors without a version counter
        other = tc.DeviceFeatureCache(10, 64, 32, DEV)
        other.write([1], x[:1])
        assert torch.equal(other.read([1], out_buffer=torch.empty(1, 64, dtype=torch.bfloat16, device=DEV)), cache.read([0]))


@pytest.mark.parametrize("aligned", [True, False])
def test_buffers_decoded_into_before_the_backward_pass_are_reported(aligned):
    buf = torch.empty(16 * 64 + 1, dtype=torch.bfloat16, device=DEV)[0 if aligned else 1:][:1024].view(16, 64)
    x = torch.randn(16, 64, device=DEV)
    codes, scales, shape = tc.quantize_mxfp4(x)
    cache = tc.DeviceFeatureCache(16, 64, 32, DEV)
    cache.write(range(16), x)
    w = torch.randn(8, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    for fill in (lambda: tc.dequantize_mxfp4(codes, scales, shape, out_buffer=buf), lambda: cache.read(range(16), out_buffer=buf)):
        y = fill() @ w.t()
        fill()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, [w], torch.ones_like(y))


@pytest.mark.parametrize("mode", ["no_grad", "inference_mode", "frozen", "reentrant"])
def test_without_a_graph_no_codes_are_made(mode, monkeypatch):
    """Evaluation of a trainable layer: only the product, and no memory but the output's."""
    from torch.utils.checkpoint import checkpoint

    from tensorcache_b200 import _lib

    x, w, b, dy = layer(8192, 16, 1024)      # many rows, few outputs: the codes would be the larger part
    w.requires_grad_(mode != "frozen")
    x.requires_grad_(mode == "reentrant")
    want = tc.int8_checkpoint_linear(x.detach(), w.detach(), b)
    made, real = [], _lib.lib()

    class Watch:
        def __getattr__(self, name):
            f = getattr(real, name)
            return (lambda *a: made.append(a[4]) or f(*a)) if name == "tcb_linear_forward" else f

    watch = Watch()
    monkeypatch.setattr(_lib, "lib", lambda: watch)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    if mode == "reentrant":      # the first pass records nothing, the second one does
        y = checkpoint(tc.int8_checkpoint_linear, x, w, b, use_reentrant=True)
        assert made == [None]
        y.backward(dy)
        assert made[0] is None and made[1] is not None
        close(x.grad, dy.double(), w.detach().double())
        close(w.grad, dy.double().t(), decoded(*plain.int8_encode(x.detach(), 32), 32))
    else:
        with {"no_grad": torch.no_grad, "inference_mode": torch.inference_mode, "frozen": torch.enable_grad}[mode]():
            y = tc.int8_checkpoint_linear(x, w, b)
        grown = torch.cuda.max_memory_allocated() - before
        assert made == [None] and grown < 8192 * 1024
    assert torch.equal(y.detach(), want)


@pytest.mark.parametrize("M,N,K", [(96, 48, 64), (130, 257, 96), (4000, 24, 128)])
@pytest.mark.parametrize("source", ["x", "sym", "amo"])
def test_gradients_equal_differences_of_whole_numbers(M, N, K, source):
    """Whole numbers small enough that nothing is rounded: outputs, gradients and their differences are exact, so the change
    of the loss over a step has to EQUAL the gradient times the step -- and neither 0 nor its negative would."""
    g = torch.Generator(device=DEV).manual_seed(M + N)

    def whole(shape, keep=0.5):
        v = torch.randint(0, 2, shape, generator=g, device=DEV) * 2 - 1
        return (v * (torch.rand(shape, generator=g, device=DEV) < keep)).to(torch.bfloat16)

    x, w, b = whole((M, K)), whole((N, K)), whole((N,))
    x[:, ::32], w[:, ::32] = 127, 0                # scale 1 in every group; no weight where a product would be large
    dy = whole((M, N), min(0.5, 60 / M))
    leaves = [w, b] + ([x] if source == "x" else [])
    for t in leaves:
        t.requires_grad_(True)
    q, s = x.detach().to(torch.int8), torch.ones(M * K // 32, dtype=torch.bfloat16, device=DEV)
    z = None
    if source == "amo":
        z = torch.full_like(s, 128, dtype=torch.uint8)
        q = (x.detach().int() + 128).to(torch.uint8)

    def output(w, b, x=x):
        return tc.int8_checkpoint_linear(x, w, b) if source == "x" else tc.fused_dequant_linear(q, s, w, b, zero_points=z)

    y = output(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y.detach().double(), x.detach().double() @ w.detach().double().t() + b.detach().double())
    for i, grad in enumerate(grads):
        moved = [t.detach() for t in leaves]
        step = whole(moved[i].shape)
        step[..., ::32] = 0 if moved[i].dim() == 2 else step[..., ::32]
        moved[i] = moved[i] + step                # at most 2: exact
        change = ((output(*moved).double() - y.detach().double()) * dy.double()).sum()
        slope = (grad.double() * step.double()).sum()
        assert float(change) == float(slope) and float(slope) != 0, (i, float(change), float(slope))


@pytest.mark.parametrize("N,K", [(8, 2080), (2080, 32)])
def test_layers_of_more_than_2_31_values(N, K):
    """More than 2^31 inputs, or outputs: zeros but for the last rows, whose results are checked."""
    M, tail = (1 << 20) + 3, slice(-300, None)
    xt, w, b, dyt = layer(300, N, K, N)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=DEV)
    x[tail] = xt
    dy = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV)
    dy[tail] = dyt
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = tc.int8_checkpoint_linear(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    check_device_status()
    X, W, D, Q = xt.double(), w.detach().double(), dyt.double(), decoded(*plain.int8_encode(xt, 32), 32)
    ones = torch.ones(1, 300, dtype=torch.float64, device=DEV)
    close(y[tail].detach(), X, W.t(), b.detach().double())
    assert bool((y[:1000] == b).all()) and not bool(dx[:1000].any())
    close(dx[tail], D, W)
    close(dw, D.t(), Q)
    close(db.view(1, -1), ones, D)
    del y, dx
    q, s, _ = tc.quantize_int8_g32(x.detach())
    y = tc.fused_dequant_linear(q.view(M, K), s, w, b)
    (dw2,) = torch.autograd.grad(y, [w], dy)
    check_device_status()
    close(y[tail].detach(), Q, W.t(), b.detach().double())
    assert bool((y[:1000] == b).all()) and torch.equal(dw2, dw)
