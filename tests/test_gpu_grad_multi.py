"""The gradient norm over many tensors and clipping by it, in 64 bits.

With u = 2^-24: a product g * grad_scale is off by u relative, so is the norm
(its squares and their sum are 64-bit), and its rounding to F32 adds u: 2u. The
coefficient adds the sum norm + 1e-6 and the division (4u together), an output
its two products (6u) and, as BF16, a rounding of 2^-8.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
WIDE = 1.01


def tensors(seed, sizes, dtypes, std=1e-2):
    g = torch.Generator("cuda").manual_seed(seed)
    return [(torch.randn(n, device="cuda", generator=g) * std).to(dtypes[i % len(dtypes)])
            for i, n in enumerate(sizes)]


def norm64(grads, scale=1.0):
    return math.sqrt(sum(float((g.double() * scale).square().sum()) for g in grads))


def check(norm, outs, grads, scale, max_norm):
    want = norm64(grads, scale)
    assert abs(norm.item() - want) <= WIDE * 2 * U * want + 1e-45
    c = min(1.0, max_norm / (want + 1e-6))
    for o, g in zip(outs, grads):
        w = g.double() * scale * c
        bound = WIDE * (6 * U + (2.0 ** -8 if o.dtype == BF16 else 0)) * w.abs() + 1e-38
        assert bool(((o.double() - w).abs() <= bound).all())


LISTS = [[1], [4095], [4096], [4097], [784 * 128, 128, 1280, 10], [1, 17, 5, 1 << 20, 0, 3],
         [100] * 48, [100] * 49, [33] * 1024, [33] * 1025, [7] * 2500, [3_000_001, 12]]


@pytest.mark.parametrize("sizes", LISTS)
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16)])
@pytest.mark.parametrize("max_norm", [1e-2, 1e6])
def test_clip(cuda, sizes, dtypes, max_norm):
    from magma_b200 import ops
    for scale in (1.0, 0.125):
        grads = tensors(1, sizes, dtypes)
        ref = [g.clone() for g in grads]
        assert ops.grad_norm_multi(grads, grad_scale=scale).item() == pytest.approx(
            norm64(ref, scale), rel=WIDE * 2 * U)
        for t in (F32, BF16):  # into other tensors, the gradients stay
            outs = [torch.empty_like(g, dtype=t) for g in grads]
            check(ops.clip_grad_norm(grads, max_norm, grad_scale=scale, out=outs), outs, ref, scale,
                  max_norm)
            assert all(torch.equal(a, b) for a, b in zip(grads, ref))
        norm = ops.clip_grad_norm(grads, max_norm, grad_scale=scale)  # in place
        check(norm, grads, ref, scale, max_norm)


def test_views_off_their_alignment(cuda):
    from magma_b200 import ops
    flat = torch.randn(50000, device="cuda")
    for dtype in (F32, BF16):
        base = flat.to(dtype)
        views = [base[1:9000], base[9003:9004], base[9006:30001], base[30004:50000]]
        ref = [v.clone() for v in views]
        around = base.clone()
        norm = ops.clip_grad_norm(views, 1.0)
        check(norm, views, ref, 1.0, 1.0)
        for i in (0, 9000, 9001, 9002, 9004, 9005, 30001, 30002, 30003):
            assert base[i] == around[i]


def test_large_and_small_values(cuda):
    """Squares beyond F32's range on both sides."""
    from magma_b200 import ops
    for size in (1e30, 1e-30):
        g = [torch.full((1000,), size, device="cuda"), torch.full((24,), size, device="cuda")]
        want = norm64(g)
        assert abs(ops.grad_norm_multi(g).item() - want) <= 2 * U * want
    zero = [torch.zeros(100, device="cuda")]
    assert ops.clip_grad_norm(zero, 1.0).item() == 0.0 and bool((zero[0] == 0).all())


def test_infinity_and_nan(cuda):
    """As the reference's mask: an infinite norm gives c = 0, a NaN norm c = 1."""
    from magma_b200 import ops
    g = [torch.ones(10, device="cuda"), torch.tensor([1.0, math.inf], device="cuda")]
    n = ops.clip_grad_norm(g, 1.0)
    assert math.isinf(n.item()) and bool((g[0] == 0).all()) and math.isnan(g[1][1].item())
    g = [torch.ones(10, device="cuda"), torch.tensor([1.0, math.nan], device="cuda")]
    n = ops.clip_grad_norm(g, 1.0)
    assert math.isnan(n.item()) and bool((g[0] == 1).all()) and math.isnan(g[1][1].item())


def test_same_bits_as_the_arena_step(cuda):
    """Clipping a list, then Adam on it, is the clipped Adam of one arena."""
    from magma_b200 import ops
    sizes = [784 * 128, 128, 1280, 10]
    arena = torch.randn(sum(sizes), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    norm = ops.grad_norm_multi(arena.split(sizes))
    p1 = torch.randn_like(arena)
    p2 = [x.clone() for x in p1.split(sizes)]
    zeros = lambda: [torch.zeros(n, device="cuda") for n in sizes]  # noqa: E731
    m, v = torch.zeros_like(arena), torch.zeros_like(arena)
    ops.adam_step_clipped(p1, arena, m, v, step=1, lr=1e-3, grad_norm=norm, max_norm=1.0)
    grads = list(arena.clone().split(sizes))
    assert torch.equal(ops.clip_grad_norm(grads, 1.0), norm)
    ops.adam_step_multi(p2, grads, zeros(), zeros(), step=1, lr=1e-3)
    assert torch.equal(torch.cat(p2), p1)


def test_front_end_refuses(cuda):
    from magma_b200 import lib, ops
    a = torch.ones(4, 6, device="cuda")
    for call in (lambda: ops.clip_grad_norm([a.t()], 1.0),
                 lambda: ops.clip_grad_norm([a], 1.0, out=[torch.ones(24, device="cuda")]),
                 lambda: ops.clip_grad_norm([a], 1.0, norm=torch.ones(2, device="cuda")),
                 lambda: ops.grad_norm_multi([])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.grad_norm_multi([a.half()])
    for call in (lambda: ops.clip_grad_norm([a, a], 1.0),
                 lambda: ops.clip_grad_norm([a, a[1:]], 1.0),
                 lambda: ops.clip_grad_norm([a], 0.0),
                 lambda: ops.clip_grad_norm([a], -1.0)):
        with pytest.raises(lib.MagmaError):
            call()
    ops.grad_norm_multi([a, a])  # reading twice is fine


def test_captured_graph(cuda):
    from magma_b200 import ops
    sizes = [5000, 3, 70000]
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        grads = tensors(5, sizes, (F32,))
        outs = [torch.empty_like(g) for g in grads]
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            norm = ops.clip_grad_norm(grads, 1.0, out=outs)
        for seed in (6, 7):
            for dst, src in zip(grads, tensors(seed, sizes, (F32,))):
                dst.copy_(src)
            g.replay()
            st.synchronize()
            check(norm, outs, grads, 1.0, 1.0)
