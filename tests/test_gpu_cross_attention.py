"""Cross attention against its definition in 64 bits.

Bounds. u = eps / 2 of a type (F32 2^-24, BF16 2^-8) is the largest relative
error of one rounding. They are first-order sums of what each step may be off,
formed elementwise in 64 bits from the inputs and widened by 5% for the products
of errors:

  score s_ij          ds = u32 (D + 4) scale sum_d |q_d||k_d|, with 2^-21 for
                      the exponential's own error and its argument's
  probability         relative 2 ds + n u32 (the sum of n terms), and u for its
                      rounding to the tensor's type before P V
  O                   sum_j (error of P_ij) |v_j| + n u32 sum P|v| + u |O|
  lse                 ds + n u32 + u32 |lse|
  dP, delta           D u32 sum |dO||V|; D u32 sum |dO||O| + sum |dO| (error of O)
  dS = P (dP - delta) P (e_P (|dP| + |delta|) + e_dP + e_delta + u |dP - delta|)
  dQ, dK, dV          the same error through the last sum, its own additions and
                      the output's rounding
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
WIDE = 1.05


def make(seed, b, h, g, m, n, d, dtype, lens=None, layout="heads", poison=True, std=1.0):
    """q, k, v, dO and the lengths; keys behind a length hold NaN and infinity."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def t(heads, length):
        x = torch.randn(b, length, heads, d, device="cuda", generator=gen) * std
        if layout == "heads":  # contiguous [B, H, S, D]
            return x.to(dtype).transpose(1, 2).contiguous()
        if layout == "tokens":  # a view of [B, S, H, D]
            return x.to(dtype).transpose(1, 2)
        # a view at an odd offset of wider rows
        wide = torch.zeros(b * length * heads * (d + 3) + 1, device="cuda", dtype=dtype)
        y = wide[1:].view(b, length, heads, d + 3)[..., 1:d + 1]
        y.copy_(x)
        return y.transpose(1, 2)

    q, k, v, do = t(h, m), t(g, n), t(g, n), t(h, m)
    if lens is not None:
        for i, e in enumerate(lens):
            if poison and e < n:
                k[i, :, e:] = float("nan")
                v[i, :, e:] = float("inf")
        lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return q, k, v, do, lens


def reference(q, k, v, do, lens, scale):
    """O, lse, dQ, dK, dV in 64 bits and how far each may be off."""
    b, h, m, d = q.shape
    g, n = k.shape[1], k.shape[2]
    u = UNIT[q.dtype]
    group = h // g
    dev = q.device
    at = torch.arange(n, device=dev)
    ends = torch.full((b,), n, device=dev) if lens is None else lens.long()
    keep = (at[None] < ends[:, None])[:, None, :, None]
    q, do = q.double(), do.double()
    k = torch.where(keep, k.double(), 0.0).repeat_interleave(group, 1)
    v = torch.where(keep, v.double(), 0.0).repeat_interleave(group, 1)
    mask = keep.transpose(-1, -2)
    t = lambda x: x.transpose(-1, -2)  # noqa: E731
    s = (q @ t(k)) * scale
    s = s.masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(mask, torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[..., None]), 0.0)
    o = p @ v
    nk = ends.double()[:, None, None, None]
    # forward
    ds_ = U32 * (d + 4) * scale * (q.abs() @ t(k.abs()))
    es = torch.where(mask, ds_, 0.0)
    worst = es.amax(-1, keepdim=True)
    ep = 2 * worst + nk * U32 + 2.0 ** -21          # relative, of a probability
    o_abs = p @ v.abs()
    eo = (ep + nk * U32 + u) * o_abs + u * o.abs() + 2 * U32 * o_abs
    el = worst[..., 0] + nk[..., 0] * U32 + 2.0 ** -22 * (1 + torch.where(lse.isinf(), 0.0, lse).abs())
    # backward; P comes from lse, which is off by el
    dp = do @ t(v)
    delta = (p * dp).sum(-1, keepdim=True)
    ep = es + el[..., None] + 2.0 ** -21
    edp = d * U32 * (do.abs() @ t(v.abs()))
    edelta = d * U32 * (do.abs() * o.abs()).sum(-1, keepdim=True) + (do.abs() * eo).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    eds = p * (ep * (dp.abs() + delta.abs()) + edp + edelta + (u + 3 * U32) * (dp - delta).abs())
    dq = scale * (ds @ k)
    edq = scale * ((eds + (nk + 2) * U32 * ds.abs()) @ k.abs()) + u * dq.abs()
    rows = m * group

    def shared(x):
        return x.reshape(b, g, group, n, d).sum(2)

    dk = shared(scale * (t(ds) @ q))
    edk = shared(scale * (t(eds + (rows + 2) * U32 * ds.abs()) @ q.abs())) + u * dk.abs()
    dv = shared(t(p) @ do)
    edv = shared(t(p * (ep + u + (rows + 2) * U32)) @ do.abs()) + u * dv.abs()
    return (o, lse, dq, dk, dv), tuple(WIDE * e + 1e-30 for e in (eo, el, edq, edk, edv))


def check(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), what  # -inf of rows without keys
    assert bool(torch.isfinite(got[fine]).all()), f"{what}: not finite"
    if fine.any():
        worst = ((got - want).abs() / bound)[fine].max().item()
        assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def run_both(case, dtype, layout="heads", seed=0, lens=None, scale=None, std=1.0):
    from magma_b200 import ops
    b, h, g, m, n, d = case
    q, k, v, do, lens = make(seed, b, h, g, m, n, d, dtype, lens, layout, std=std)
    scale = d ** -0.5 if scale is None else scale
    want, bound = reference(q, k, v, do, lens, scale)
    o, lse = ops.cross_attention_fwd(q, k, v, scale, lens)
    check(o, want[0], bound[0], "o")
    check(lse, want[1], bound[1], "lse")
    grads = ops.cross_attention_bwd(q, k, v, o, do, lse, scale, lens)
    for x, w, e, name in zip(grads, want[2:], bound[2:], ("dq", "dk", "dv")):
        check(x, w, e, name)
    assert ops.device_error_check() == 0
    return (q, k, v, do, lens), o, lse, grads


# sizes around the tiles of 16, 64 and 128 rows and keys, head sizes that are
# and are not multiples of 8 and 64, shared heads
SIZES = [
    (1, 1, 1, 1, 1, 1), (1, 2, 1, 1, 7, 8), (2, 2, 2, 5, 63, 32), (1, 3, 3, 64, 64, 64),
    (2, 4, 2, 65, 127, 64), (1, 2, 1, 127, 129, 128), (1, 2, 2, 128, 128, 128),
    (1, 6, 2, 129, 257, 64), (2, 4, 1, 33, 300, 80), (1, 8, 2, 40, 191, 96), (1, 2, 2, 17, 65, 17),
    (3, 2, 1, 200, 333, 72), (1, 5, 5, 256, 384, 64), (1, 4, 4, 300, 513, 128),
    (1, 16, 2, 2, 130, 128), (2, 12, 4, 3, 1025, 64),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", SIZES)
def test_matches_the_definition(cuda, case, dtype):
    run_both(case, dtype)


# lengths: none, one, tile borders and one off, all; NaN and infinity behind them
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case,lens", [
    ((4, 2, 1, 70, 130, 64), [0, 1, 64, 130]), ((4, 4, 2, 130, 300, 128), [127, 128, 129, 300]),
    ((3, 2, 2, 1, 200, 64), [0, 1, 199]), ((3, 4, 1, 2, 257, 128), [256, 0, 65]),
    ((2, 2, 1, 40, 40, 48), [0, 0]), ((3, 6, 2, 150, 600, 64), [511, 513, 2]),
    ((2, 3, 3, 20, 129, 33), [63, 128]),
])
def test_lengths_and_what_lies_behind_them(cuda, case, lens, dtype):
    run_both(case, dtype, lens=lens)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("case,lens", [
    ((2, 4, 2, 70, 131, 64), [131, 40]), ((2, 4, 4, 1, 90, 128), [17, 90]),
    ((1, 2, 2, 140, 200, 128), None),
])
def test_strides(cuda, case, lens, layout, dtype):
    run_both(case, dtype, layout=layout, lens=lens)


# one query and a few queries over sources that are split over the GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(1, 8, 8, 1, 5000, 64), (1, 8, 1, 1, 4097, 128),
                                  (2, 8, 2, 4, 3001, 128), (1, 2, 2, 100, 6000, 64),
                                  (1, 32, 1, 1, 2000, 64), (5, 4, 2, 1, 1, 80)])
def test_few_queries_over_long_sources(cuda, case, dtype):
    run_both(case, dtype)


# few tiles with many steps: the gradient's steps are dealt out over the GPU and
# units are put together from pieces, also next to sequences without keys
@pytest.mark.parametrize("case,lens", [
    ((1, 4, 1, 520, 300, 64), None), ((2, 8, 2, 450, 200, 128), [200, 77]),
    ((3, 2, 1, 130, 2100, 64), [2100, 0, 1999]), ((2, 4, 4, 260, 1900, 128), [1, 1900]),
    ((1, 2, 2, 1700, 2200, 80), None), ((5, 3, 1, 600, 700, 64), [0, 700, 64, 129, 500]),
    ((1, 1, 1, 65, 9000, 128), None), ((4, 6, 2, 700, 1664, 96), [1664, 1000, 128, 1663]),
])
def test_gradient_with_steps_dealt_out(cuda, case, lens):
    first = run_both(case, torch.bfloat16, lens=lens)
    again = run_both(case, torch.bfloat16, lens=lens)
    for a, b in zip(first[3], again[3]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale,std", [(0.0, 1.0), (1.0, 2.0), (1e-3, 30.0)])
def test_scales(cuda, scale, std, dtype):
    run_both((1, 2, 1, 90, 140, 64), dtype, scale=scale, std=std)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores_stay_finite(cuda, dtype):
    """Scores of several thousand: the running maximum keeps the exponentials in range."""
    from magma_b200 import ops
    for m in (1, 130):
        q, k, v, do, _ = make(3, 1, 2, 2, m, 200, 64, dtype)
        o, lse = ops.cross_attention_fwd(q * 30, k * 30, v, 1.0)
        s = (q * 30).double() @ (k * 30).double().transpose(-1, -2)
        assert (lse.double() - torch.logsumexp(s, -1)).abs().max() <= 1e-5 * s.abs().max()
        assert bool(torch.isfinite(o.float()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_broadcast_inputs(cuda, dtype):
    """One source for all sequences, one gradient for all positions (strides of 0)."""
    from magma_b200 import ops
    q, k, v, do, _ = make(5, 3, 4, 2, 66, 130, 64, dtype)
    k1, v1 = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)
    d1 = do[:, :, :1].expand(-1, -1, 66, -1)
    want, bound = reference(q, k1, v1, d1, None, 0.125)
    o, lse = ops.cross_attention_fwd(q, k1, v1, 0.125)
    check(o, want[0], bound[0], "o")
    for x, w, e in zip(ops.cross_attention_bwd(q, k1, v1, o, d1, lse, 0.125), want[2:], bound[2:]):
        check(x, w, e, "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_given_outputs_and_their_neighbours(cuda, dtype):
    """Outputs inside wider tensors: what lies around them stays as it was."""
    from magma_b200 import ops
    b, h, g, m, n, d = 2, 4, 2, 70, 90, 64
    q, k, v, do, _ = make(6, b, h, g, m, n, d, dtype)
    lens = torch.tensor([90, 33], dtype=torch.int32, device="cuda")

    def inside(heads, length):
        whole = torch.full((b, length + 5, heads, d + 8), 7.0, device="cuda", dtype=dtype)
        return whole, whole[:, :length, :, :d].transpose(1, 2)

    (wo, o), (wq, dq), (wk, dk), (wv, dv) = (inside(*x) for x in ((h, m), (h, m), (g, n), (g, n)))
    _, lse = ops.cross_attention_fwd(q, k, v, 0.125, lens, out=o)
    ops.cross_attention_bwd(q, k, v, o, do, lse, 0.125, lens, dq=dq, dk=dk, dv=dv)
    want, bound = reference(q, k, v, do, lens, 0.125)
    for x, w, e in zip((o, dq, dk, dv), (want[0], *want[2:]), (bound[0], *bound[2:])):
        check(x, w, e, "output")
    for whole, inner in ((wo, o), (wq, dq), (wk, dk), (wv, dv)):
        inner.fill_(7.0)
        assert bool((whole == 7.0).all())


def test_bad_lengths_are_clamped_and_reported(cuda):
    from magma_b200 import lib, ops
    q, k, v, _, _ = make(7, 2, 2, 2, 3, 20, 64, torch.bfloat16)
    lens = torch.tensor([-3, 99], dtype=torch.int32, device="cuda")
    o, lse = ops.cross_attention_fwd(q, k, v, 0.125, lens)
    with pytest.raises(lib.MagmaError):
        ops.device_error_check()
    assert ops.device_error_check() == 0
    ok = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    o2, lse2 = ops.cross_attention_fwd(q, k, v, 0.125, ok)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_front_end_refuses(cuda):
    from magma_b200 import lib, ops
    q, k, v, do, _ = make(8, 2, 4, 2, 6, 10, 64, torch.float32)
    with pytest.raises(TypeError):
        ops.cross_attention_fwd(q, k.bfloat16(), v)
    with pytest.raises(TypeError):
        ops.cross_attention_fwd(q.half(), k.half(), v.half())
    with pytest.raises(ValueError):
        ops.cross_attention_fwd(q, k, v[:, :, :5])
    with pytest.raises(ValueError):
        ops.cross_attention_fwd(q, k[:1], v[:1])
    with pytest.raises(ValueError):
        ops.cross_attention_fwd(q.transpose(2, 3), k, v)
    with pytest.raises(ValueError):
        ops.cross_attention_fwd(q, k, v, kv_lens=torch.tensor([1, 2], device="cuda"))
    with pytest.raises(lib.MagmaError):
        ops.cross_attention_fwd(q, k, v, out=torch.empty_like(q[:, :1]).expand(-1, 4, -1, -1))
    with pytest.raises(lib.MagmaError):
        ops.cross_attention_fwd(q[:, :3], k, v)
    o, lse = ops.cross_attention_fwd(q, k, v)
    with pytest.raises(ValueError):
        ops.cross_attention_bwd(q, k, v, o, do, lse.double())
    with pytest.raises(ValueError):
        ops.cross_attention_bwd(q, k, v, o, do[:, :2], lse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_queries_or_no_keys(cuda, dtype):
    """Nothing to attend with: dK and dV are 0. Nothing to attend to: O and dQ are 0."""
    from magma_b200 import ops
    q, k, v, do, _ = make(12, 2, 4, 2, 5, 9, 64, dtype)
    none = q[:, :, :0]
    o, lse = ops.cross_attention_fwd(none, k, v)
    assert o.shape == none.shape and lse.shape == none.shape[:3]
    _, dk, dv = ops.cross_attention_bwd(none, k, v, o, o, lse)
    assert bool((dk == 0).all()) and bool((dv == 0).all())
    o, lse = ops.cross_attention_fwd(q, k[:, :, :0], v[:, :, :0])
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, _ = ops.cross_attention_bwd(q, k[:, :, :0], v[:, :, :0], o, do, lse)
    assert bool((dq == 0).all()) and dk.shape[2] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(2, 4, 2, 1, 3000, 64), (1, 2, 1, 90, 4000, 128),
                                  (2, 4, 4, 3, 500, 64), (1, 2, 2, 600, 64, 64)])
def test_smaller_workspaces(cuda, case, dtype):
    """The forward pass takes any workspace; the gradient refuses one that is too small."""
    import ctypes as C

    from magma_b200 import lib, ops
    b, h, g, m, n, d = case
    q, k, v, do, _ = make(13, b, h, g, m, n, d, dtype)
    want, bound = reference(q, k, v, do, None, d ** -0.5)
    dt = lib.F32 if dtype == torch.float32 else lib.BF16
    keep = []

    def st(t):
        keep.append((C.c_int64 * 3)(*t.stride()[:3]))
        return C.addressof(keep[-1])

    need = lib.query("magma_cross_attention_fwd_workspace_size", b, h, g, m, n, d, dt)
    for size in {0, 16, need // 3 // 16 * 16, need, need + 4096}:
        ws = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
        o, lse = torch.empty_like(q), torch.empty(b, h, m, device="cuda")
        lib.call("magma_cross_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                 lse.data_ptr(), None, b, h, g, m, n, d, st(q), st(k), st(v), st(o), d ** -0.5, dt,
                 ws.data_ptr() if size else None, size, torch.cuda.current_stream().cuda_stream)
        check(o, want[0], bound[0], "o")
        check(lse, want[1], bound[1], "lse")
    need = lib.query("magma_cross_attention_bwd_workspace_size", b, h, g, m, n, d, dt)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]

    def bwd(size):
        lib.call("magma_cross_attention_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                 do.data_ptr(), lse.data_ptr(), None, *[t.data_ptr() for t in grads], b, h, g, m, n,
                 d, st(q), st(k), st(v), st(o), st(do), *[st(t) for t in grads], d ** -0.5, dt,
                 ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)

    with pytest.raises(lib.MagmaError):
        bwd(need - 16)
    bwd(need)
    for x, w, e in zip(grads, want[2:], bound[2:]):
        check(x, w, e, "gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 150])
def test_captured_graphs_and_streams(cuda, m, dtype):
    """Two captured graphs and eager calls on two streams at once, on new inputs."""
    from magma_b200 import ops
    sets = [make(20 + i, 2, 4, 2, m, 700, 64, dtype, [700, 300], poison=False) for i in range(4)]

    def step(s):
        o, lse = ops.cross_attention_fwd(*s[:3], 0.125, s[4])
        return (o, lse) + ops.cross_attention_bwd(*s[:3], o, s[3], lse, 0.125, s[4])

    want = [step(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs, statics = [], [], []
    for st in streams:
        static = [x.clone() for x in sets[0]]
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                out = step(static)
        graphs.append(g), outs.append(out), statics.append(static)
    for i in range(2):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                for dst, src in zip(statics[j], sets[2 * i + j]):
                    dst.copy_(src)
                graphs[j].replay()
        with torch.cuda.stream(streams[0]):
            eager = step(sets[3])
        torch.cuda.synchronize()
        for j in range(2):
            for a, b in zip(outs[j], want[2 * i + j]):
                assert torch.equal(a, b)
        for a, b in zip(eager, want[3]):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(cuda):
    """A sequence that starts more than 2^31 elements into the cache."""
    from magma_b200 import ops
    far = (1 << 31) + 64
    pool = torch.zeros(far + 8192, dtype=torch.bfloat16, device="cuda")
    q, k, v, do, _ = make(9, 2, 2, 1, 1, 60, 64, torch.bfloat16)
    kk = pool.as_strided((2, 1, 60, 64), (far, 60 * 64, 64, 1))
    kk.copy_(k)
    for m in (1, 100):
        q, _, _, do, _ = make(9, 2, 2, 1, m, 60, 64, torch.bfloat16)
        want, bound = reference(q, k, v, do, None, 0.125)
        o, lse = ops.cross_attention_fwd(q, kk, v, 0.125)
        check(o, want[0], bound[0], "o")
        dk = pool.as_strided((2, 1, 60, 64), (far, 60 * 64, 64, 1), 3840)
        ops.cross_attention_bwd(q, kk, v, o, do, lse, 0.125, dk=dk)
        check(dk, want[3], bound[3], "dk")


def test_gradient_against_differences(cuda):
    """<dq, e> for a direction e against central differences of the definition.

    sum(O dO) along q + t e, k + t e', v + t e'' is analytic in t; with t = 1e-3 the
    difference quotient's error t^2 f'''/6 is measured by halving t (Richardson:
    a third of what the two quotients differ by bounds it fourfold)."""
    from magma_b200 import ops
    q, k, v, do, lens = make(11, 2, 4, 2, 40, 70, 64, torch.float32, [70, 31], poison=False)
    want, bound = reference(q, k, v, do, lens, 0.125)
    o, lse = ops.cross_attention_fwd(q, k, v, 0.125, lens)
    grads = ops.cross_attention_bwd(q, k, v, o, do, lse, 0.125, lens)
    dirs = [torch.randn(x.shape, device="cuda", dtype=torch.float64,
                        generator=torch.Generator("cuda").manual_seed(i)) for i, x in enumerate((q, k, v))]

    def f(t):
        x = [a.double() + t * e for a, e in zip((q, k, v), dirs)]
        at = torch.arange(70, device="cuda")
        mask = (at[None] < lens[:, None])[:, None, None, :]
        s = (x[0] @ x[1].repeat_interleave(2, 1).transpose(-1, -2) * 0.125).masked_fill(~mask, -math.inf)
        return ((torch.softmax(s, -1) @ x[2].repeat_interleave(2, 1)) * do.double()).sum().item()

    quot = [(f(t) - f(-t)) / (2 * t) for t in (1e-3, 5e-4)]
    got = sum((g.double() * e).sum().item() for g, e in zip(grads, dirs))
    off = sum((b * e.abs()).sum().item() for b, e in zip(bound[2:], dirs))
    assert abs(got - quot[1]) <= off + 4 * abs(quot[0] - quot[1]) / 3 + 1e-9 * abs(quot[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_key_reaches_every_row(dtype, d):
    """A NaN in a key that counts makes its scores NaN, whichever column of a tile
    it is in, and with them the rows of its heads; other heads stay finite."""
    from magma_b200 import ops
    q, k, v, do, _ = make(77, 1, 8, 8, 130, 200, d, dtype)
    clean, _ = ops.cross_attention_fwd(q, k, v)
    for h in range(8):
        k[0, h, 128 + h, 0] = float("nan")
    k[0, 7, 135, 0] = 0.5
    o, lse = ops.cross_attention_fwd(q, k, v)
    assert torch.isnan(o[0, :7]).all() and torch.isnan(lse[0, :7]).all()
    assert torch.isfinite(o[0, 7]).all()
    for h in range(8):
        k[0, h, 128 + h, 0] = 0.5
        k[0, h, h, 0] = float("nan")
    o, lse = ops.cross_attention_fwd(q, k, v)
    assert torch.isnan(o).all() and torch.isnan(lse).all()
    assert torch.isfinite(clean).all()


@pytest.mark.parametrize("case", [(2, 4, 2, 9, 8, 128), (1, 4, 1, 133, 20, 64), (5, 4, 4, 7, 81, 32),
                                  (2, 6, 2, 40, 453, 96), (1, 2, 2, 115, 691, 32)])
def test_small_gradients_have_the_error_of_their_rounding(cuda, case):
    """Relative RMS error against that of rounding the exact gradient. P and dS reach the
    products to 2^-17, so what is left is the rounding of the stored O in delta: relative
    to dP it is sqrt(sum P^2) of a rounding, at most 0.2 for 64 keys and more of unit
    scores (sum P^2 = e / n), and no part of it where all keys are in one tile.
    sqrt(1 + 0.2^2) = 1.02; the RMS of 2000 roundings scatters by 1 / sqrt(2000) = 2% of
    itself, three of those and the few dominant elements of a short source make 1.15."""
    from magma_b200 import ops
    b, h, g, m, n, d = case
    q, k, v, do, _ = make(91, b, h, g, m, n, d, torch.bfloat16)
    o, lse = ops.cross_attention_fwd(q, k, v)
    got = ops.cross_attention_bwd(q, k, v, o, do, lse)
    x, y, z = (t.double().requires_grad_() for t in (q, k, v))
    s = x @ y.repeat_interleave(h // g, 1).transpose(2, 3) * d ** -0.5
    (s.softmax(-1) @ z.repeat_interleave(h // g, 1)).backward(do.double())
    for name, a, want in zip(("dq", "dk", "dv"), got, (x.grad, y.grad, z.grad)):
        err = (a.double() - want).norm()
        least = (want.to(torch.bfloat16).double() - want).norm()
        assert err <= 1.15 * least, (name, (err / least).item())


# more sequences than the tables of lengths and steps hold, and than a warp ranks
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(600, 2, 1, 40, 150, 64), (300, 2, 2, 30, 100, 128),
                                  (512, 1, 1, 70, 200, 32), (33, 4, 2, 65, 130, 64)])
def test_many_sequences(cuda, case, dtype):
    b, n = case[0], case[4]
    run_both(case, dtype, lens=[(37 * i) % (n + 1) for i in range(b)])
    if b == 600:
        run_both(case, dtype)


def test_gradients_back_to_back(cuda):
    """The launches of a call overlap at their ends, those of two calls do not: calls
    that follow one another on other inputs, in memory that the ones before gave back,
    find the same bits. Short sources, whose delta comes from dQ, are among them."""
    from magma_b200 import ops
    sets = [make(s, 8, 8, 4, 200, 400, 64, torch.bfloat16, lens=lens)
            for s, lens in ((1, [400, 3, 64, 65, 0, 333, 40, 128]), (2, [64] * 8), (3, None))]

    def gradients(i):
        q, k, v, do, lens = sets[i]
        o, lse = ops.cross_attention_fwd(q, k, v, kv_lens=lens)
        return ops.cross_attention_bwd(q, k, v, o, do, lse, kv_lens=lens)

    first = []
    for i in range(len(sets)):
        first.append([x.clone() for x in gradients(i)])
        torch.cuda.synchronize()
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for turn in range(60):
        for x, y in zip(gradients(turn % 3), first[turn % 3]):
            wrong += (x != y).sum()
    assert int(wrong) == 0
