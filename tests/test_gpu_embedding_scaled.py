"""The scaled embedding lookup and its gradient against their definitions in 64 bits.

u = eps / 2 of a type bounds one rounding. A lookup rounds the product and the
sum in F32, and once more to a BF16 output. A gradient row adds n values in F32
(at most n u32 times the sum of their sizes off), multiplies by the scale, adds
to what was there, and rounds to the output's type.
"""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
UNIT = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}
WIDE = 1.01
F32, BF16 = torch.float32, torch.bfloat16


def check(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    assert bool((off <= WIDE * bound).all()), f"{what}: {(off / (bound + 1e-300)).max().item():.3g} times the bound"


def batch(seed, b, n, d, v, dtype, kind="any"):
    g = torch.Generator("cuda").manual_seed(seed)
    if kind == "one":
        tok = torch.full((b, n), v - 1, device="cuda")
    elif kind == "few":
        tok = torch.randint(0, min(v, 3), (b, n), device="cuda", generator=g)
    else:
        tok = torch.randint(0, v, (b, n), device="cuda", generator=g)
    dout = torch.randn(b * n, d, device="cuda", generator=g).to(dtype)
    return tok.int(), dout


@pytest.mark.parametrize("ti,to", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("b,n,d,v,with_pos", [
    (1, 1, 1, 1, True), (2, 3, 8, 5, False), (1, 17, 777, 100, True), (4, 33, 512, 1000, True),
    (2, 5, 1032, 50, False), (3, 1, 2048, 7, True), (16, 1, 512, 32000, True),
])
def test_lookup(cuda, b, n, d, v, with_pos, ti, to):
    from magma_b200 import ops
    tok, _ = batch(1, b, n, d, v, F32)
    table = torch.randn(v, d, device="cuda").to(ti)
    pos = torch.randn(n + 2, d, device="cuda").to(ti) if with_pos else None
    scale = d ** 0.5
    got = ops.embedding_scaled_fwd(tok, table, pos, scale=scale, out_dtype=to)
    assert got.dtype == to
    rows = table.double()[tok.reshape(-1).long()] * scale
    want = rows + (pos[:n].double().repeat(b, 1) if with_pos else 0.0)
    # the scale itself reaches the kernel rounded to F32
    check(got, want, U32 * (2 * rows.abs() + want.abs()) + UNIT[to] * want.abs(), "lookup")
    assert ops.device_error_check() == 0


def test_lookup_of_strided_and_odd_tables(cuda):
    from magma_b200 import ops
    tok, _ = batch(2, 2, 9, 64, 20, F32)
    whole = torch.randn(20, 100, device="cuda")
    for view in (whole[:, :64], whole[:, 1:65], whole[:, 4:68]):
        got = ops.embedding_scaled_fwd(tok, view, scale=2.0)
        assert torch.equal(got, view[tok.reshape(-1).long()] * 2.0)
    out = torch.full((20, 64), 7.0, device="cuda")
    ops.embedding_scaled_fwd(tok, whole[:, :64], scale=1.0, out=out[1:19])
    assert bool((out[0] == 7).all() and (out[19] == 7).all())
    assert torch.equal(out[1:19], whole[:, :64][tok.reshape(-1).long()])


def gradient_reference(tok, dout, v, scale, pad, old=None):
    t = tok.reshape(-1).long()
    x = dout.double()
    if pad is not None:
        x = torch.where((t != pad)[:, None], x, 0.0)
    zero = torch.zeros(v, x.shape[1], dtype=torch.float64, device="cuda")
    total, size = zero.index_add(0, t, x), zero.index_add(0, t, x.abs())
    count = torch.bincount(t, minlength=v).double()[:, None]
    want = total * scale
    bound = count * U32 * size * scale + 2 * U32 * want.abs()
    if old is not None:
        want = want + old.double()
        bound = bound + U32 * want.abs()
    return want, bound


CASES = [(1, 1, 1, 1, "any"), (1, 3, 8, 4, "any"), (2, 37, 40, 11, "any"), (1, 9, 777, 30, "few"),
         (4, 64, 384, 65, "any"), (3, 300, 128, 255, "any"), (3, 300, 128, 256, "any"),
         (2, 1100, 64, 70000, "any"), (1, 4097, 512, 50257, "any"), (8, 1024, 96, 65536, "few"),
         (1, 8193, 64, 100, "one"), (9, 1000, 72, 65535, "one"), (2, 70000, 16, 300, "any"),
         (1, 20, 1024, 20000000, "any")]


@pytest.mark.parametrize("td,tt", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("b,n,d,v,kind", CASES)
def test_gradient(cuda, b, n, d, v, kind, td, tt):
    from magma_b200 import ops
    if v > 1000000:
        d = 16
    tok, dout = batch(3, b, n, d, v, td, kind)
    dout = dout[:, :d]
    for pad in (None, 0) if kind != "one" else (None, v - 1):
        got, dpos = ops.embedding_scaled_bwd(tok, dout, v, scale=1.5, padding_idx=pad, pos=True,
                                             dtype=tt)
        want, bound = gradient_reference(tok, dout, v, 1.5, pad)
        check(got, want, bound + UNIT[tt] * want.abs(), "dtable")
        x = dout.double().reshape(b, n, d)
        check(dpos, x.sum(0), b * U32 * x.abs().sum(0), "dpos")
        again, dpos2 = ops.embedding_scaled_bwd(tok, dout, v, scale=1.5, padding_idx=pad, pos=True,
                                                dtype=tt)
        assert torch.equal(got, again) and torch.equal(dpos, dpos2)
    assert ops.device_error_check() == 0


# Small tables under many rows, long rows, and sizes around the tiles' borders.
MORE = [(16, 1024, 384, 65, "any"), (4, 2048, 1000, 192, "any"), (4, 2048, 1000, 193, "any"),
        (2, 1024, 33, 7, "few"), (2, 1025, 33, 7, "few"), (8, 512, 4800, 5, "any"), (1, 1, 31, 192, "any"),
        (1, 300, 512, 257, "few"), (2, 1000, 512, 3001, "few"), (1, 2500, 1024, 312, "any"),
        (1, 2497, 1024, 312, "any")]


@pytest.mark.parametrize("td,tt", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("b,n,d,v,kind", MORE)
def test_gradient_of_small_tables_and_long_rows(cuda, b, n, d, v, kind, td, tt):
    test_gradient(cuda, b, n, d, v, kind, td, tt)


def test_bad_tokens_of_a_small_table(cuda):
    from magma_b200 import lib, ops
    tok, dout = batch(11, 8, 1024, 640, 30, F32)
    tok[0, 5], tok[7, 1023], tok[3, 3] = -1, 30, 2 ** 31 - 1
    got, _ = ops.embedding_scaled_bwd(tok, dout, 30)
    with pytest.raises(lib.MagmaError):
        ops.device_error_check()
    t = tok.reshape(-1)
    good = (t >= 0) & (t < 30)
    want, bound = gradient_reference(t[good], dout[good], 30, 1.0, None)
    check(got, want, bound, "dtable")


@pytest.mark.parametrize("tt", [F32, BF16])
@pytest.mark.parametrize("d", [64, 77])
def test_gradient_accumulates(cuda, d, tt):
    from magma_b200 import ops
    tok, dout = batch(4, 3, 50, d, 40, F32)
    old, oldp = torch.randn(40, d, device="cuda").to(tt), torch.randn(60, d, device="cuda")
    dtable, dpos = old.clone(), oldp.clone()
    ops.embedding_scaled_bwd(tok, dout, 40, scale=2.0, padding_idx=3, dtable=dtable, dpos=dpos,
                             accumulate=True, accumulate_pos=True)
    want, bound = gradient_reference(tok, dout, 40, 2.0, 3, old)
    check(dtable, want, bound + UNIT[tt] * want.abs(), "dtable")
    assert torch.equal(dtable[3], old[3]) and torch.equal(dpos[50:], oldp[50:])
    x = dout.double().reshape(3, 50, d)
    check(dpos[:50], x.sum(0) + oldp[:50], 4 * U32 * (x.abs().sum(0) + oldp[:50].abs()), "dpos")


def test_gradient_of_strided_rows_into_a_wider_table(cuda):
    from magma_b200 import ops
    tok, wide = batch(5, 2, 33, 100, 15, F32)
    for lo in (0, 1, 4):
        dout = wide[:, lo:lo + 64]
        whole = torch.full((17, 80), 7.0, device="cuda")
        ops.embedding_scaled_bwd(tok, dout, 15, dtable=whole[1:16, lo:lo + 64])
        want, bound = gradient_reference(tok, dout, 15, 1.0, None)
        check(whole[1:16, lo:lo + 64], want, bound, "dtable")
        whole[1:16, lo:lo + 64] = 7.0
        assert bool((whole == 7.0).all())
    # one gradient row for all tokens (stride 0) is refused, not misread
    from magma_b200 import lib
    with pytest.raises(lib.MagmaError):
        ops.embedding_scaled_bwd(tok, wide[:1, :64].expand(66, 64), 15)


def test_empty_batches(cuda):
    from magma_b200 import ops
    tok = torch.zeros(0, 5, dtype=torch.int32, device="cuda")
    table = torch.randn(9, 16, device="cuda")
    assert ops.embedding_scaled_fwd(tok, table).shape == (0, 16)
    g, p = ops.embedding_scaled_bwd(tok, torch.zeros(0, 16, device="cuda"), 9, pos=True)
    assert g.shape == (9, 16) and bool((g == 0).all()) and p.shape == (5, 16) and bool((p == 0).all())


def test_bad_tokens_are_skipped_and_reported(cuda):
    from magma_b200 import lib, ops
    tok = torch.tensor([[0, 9, -1, 3]], dtype=torch.int32, device="cuda")
    table = torch.randn(5, 16, device="cuda")
    out = ops.embedding_scaled_fwd(tok, table, scale=3.0)
    with pytest.raises(lib.MagmaError):
        ops.device_error_check()
    assert bool((out[1:3] == 0).all()) and torch.equal(out[0], table[0] * 3.0)
    dout = torch.randn(4, 16, device="cuda")
    g, _ = ops.embedding_scaled_bwd(tok, dout, 5)
    with pytest.raises(lib.MagmaError):
        ops.device_error_check()
    want = torch.zeros(5, 16, device="cuda")
    want[0], want[3] = dout[0], dout[3]
    assert torch.equal(g, want)
    assert ops.device_error_check() == 0


def test_front_end_refuses(cuda):
    from magma_b200 import ops
    tok, dout = batch(6, 2, 3, 16, 5, F32)
    table = torch.zeros(5, 16, device="cuda")
    for call in (lambda: ops.embedding_scaled_fwd(tok.long(), table),
                 lambda: ops.embedding_scaled_fwd(tok[0], table),
                 lambda: ops.embedding_scaled_fwd(tok, table.t()),
                 lambda: ops.embedding_scaled_fwd(tok, table, table[:2]),
                 lambda: ops.embedding_scaled_fwd(tok, table, out=torch.zeros(5, 16, device="cuda")),
                 lambda: ops.embedding_scaled_bwd(tok, dout[:5], 5),
                 lambda: ops.embedding_scaled_bwd(tok, dout, 5, padding_idx=5),
                 lambda: ops.embedding_scaled_bwd(tok, dout, 5, dtable=table[:4])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.embedding_scaled_fwd(tok, table.half())


def test_captured_graphs_and_streams(cuda):
    from magma_b200 import ops
    sets = [batch(30 + i, 4, 500, 64, 700, F32) for i in range(2)]
    want = [ops.embedding_scaled_bwd(t, x, 700, scale=2.0, padding_idx=0, pos=True) for t, x in sets]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    tok, dout = sets[0][0].clone(), sets[0][1].clone()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = ops.embedding_scaled_bwd(tok, dout, 700, scale=2.0, padding_idx=0, pos=True)
    for i in (1, 0):
        with torch.cuda.stream(st):
            tok.copy_(sets[i][0]), dout.copy_(sets[i][1])
            g.replay()
        eager = ops.embedding_scaled_bwd(*sets[i], 700, scale=2.0, padding_idx=0, pos=True)
        torch.cuda.synchronize()
        for a, b, c in zip(out, eager, want[i]):
            assert torch.equal(a, c) and torch.equal(b, c)


def test_gradient_against_differences(cuda):
    """sum(out dOut) is linear in the table: the gradient is its difference quotient."""
    from magma_b200 import ops
    tok, dout = batch(7, 2, 40, 32, 13, F32)
    g, _ = ops.embedding_scaled_bwd(tok, dout, 13, scale=1.5)
    e = torch.randn(13, 32, device="cuda", dtype=torch.float64)
    diff = (e[tok.reshape(-1).long()] * 1.5 * dout.double()).sum()
    _, bound = gradient_reference(tok, dout, 13, 1.5, None)
    assert abs((g.double() * e).sum() - diff) <= WIDE * (bound * e.abs()).sum()
