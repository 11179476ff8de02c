"""Cross attention at its edges: values that are no ordinary numbers, and sizes of
zero. Tolerances are those of test_gpu_cross_attention."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_cross_attention import check, make, reference  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]

# Sources that are cut into parts: a few queries in chunks, query tiles too few for
# the GPU (BF16: tensor cores, F32: FMA pipe), and one that is not cut in BF16.
SPLIT = [(1, 8, 8, 1, 5000, 64), (2, 8, 2, 4, 9000, 128), (1, 2, 2, 100, 6000, 64),
         (1, 2, 1, 70, 6000, 128), (1, 8, 8, 130, 200, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SPLIT)
def test_nan_query_of_a_split_source(cuda, case, dtype):
    """Every part's scores of that row are NaN: so are its output and lse, and no
    other row's."""
    from magma_b200 import ops
    b, h, g, m, n, d = case
    q, k, v, do, _ = make(31, b, h, g, m, n, d, dtype)
    want, bound = reference(q, k, v, do, None, d ** -0.5)
    bad = torch.zeros(b, h, m, dtype=torch.bool, device="cuda")
    bad[0, h - 1, m - 1] = True
    q[bad, d - 1] = math.nan
    o, lse = ops.cross_attention_fwd(q, k, v)
    assert bool(torch.isnan(o[bad]).all()) and bool(torch.isnan(lse[bad]).all())
    check(o[~bad], want[0][~bad], bound[0][~bad], "o")
    check(lse[~bad], want[1][~bad], bound[1][~bad], "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SPLIT)
def test_nan_key_where_one_part_has_keys(cuda, case, dtype):
    """A sequence so short that only the first part has keys, one of them NaN: the
    empty parts do not make its rows those of a sequence without keys."""
    from magma_b200 import ops
    _, h, g, m, n, d = case
    q, k, v, do, lens = make(32, 3, h, g, m, n, d, dtype, [n, 20, 0])
    want, bound = reference(q, k, v, do, lens, d ** -0.5)
    k[1, 0, 3, 0] = math.nan
    o, lse = ops.cross_attention_fwd(q, k, v, kv_lens=lens)
    bad = torch.zeros(3, h, m, dtype=torch.bool, device="cuda")
    bad[1, :h // g] = True
    assert bool(torch.isnan(o[bad]).all()) and bool(torch.isnan(lse[bad]).all())
    check(o[~bad], want[0][~bad], bound[0][~bad], "o")
    check(lse[~bad], want[1][~bad], bound[1][~bad], "lse")
    assert bool((o[2] == 0).all()) and bool((lse[2] == -math.inf).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(1, 2, 2, 200, 300, 64), (1, 2, 1, 200, 300, 128),
                                  (1, 2, 2, 100, 6000, 64), (2, 4, 2, 130, 700, 96),
                                  (1, 2, 2, 3, 300, 64), (3, 40, 40, 300, 400, 64)])
def test_first_keys_score_minus_infinity(cuda, case, dtype):
    """The first 128 keys' scores are -inf, the others' about -500: the output is
    that of the other keys, however far below 0 their largest score is."""
    from magma_b200 import ops
    b, h, g, m, n, d = case
    q, k, v, do, _ = make(33, b, h, g, m, n, d, dtype)
    q[..., 0] = 1.0
    k[..., 0] = -4000.0 / 64 ** 0.5 * d ** 0.5
    k[:, :, :128, 0] = -math.inf
    want, bound = reference(q, k[:, :, 128:], v[:, :, 128:], do, None, d ** -0.5)
    o, lse = ops.cross_attention_fwd(q, k, v)
    check(o, want[0], bound[0], "o")
    check(lse, want[1], bound[1], "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,g", [(2, 0, 2), (0, 4, 2), (0, 0, 0), (2, 0, 0)])
def test_gradient_without_heads_or_sequences(cuda, b, h, g, dtype):
    """No query heads: dK and dV are 0. No sequences: nothing to write."""
    from magma_b200 import ops
    q = torch.ones(b, h, 70, 64, device="cuda", dtype=dtype)
    k = torch.ones(b, g, 200, 64, device="cuda", dtype=dtype)
    o, lse = ops.cross_attention_fwd(q, k, k)
    assert o.shape == q.shape and lse.shape == (b, h, 70)
    dk, dv = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
    dq, dk, dv = ops.cross_attention_bwd(q, k, k, o, q, lse, dk=dk, dv=dv)
    assert dq.shape == q.shape and bool((dk == 0).all()) and bool((dv == 0).all())


# every path: a few queries in a cluster, in joined chunks, in one chunk; tensor cores or
# FMA pipe whole and in parts; an odd head size
PATHS = SPLIT + [(1, 8, 8, 1, 777, 64), (2, 4, 4, 1, 20, 64), (2, 8, 8, 200, 300, 128),
                 (2, 4, 2, 150, 260, 33)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", PATHS)
@pytest.mark.parametrize("last", [False, True])
def test_an_infinite_score(cuda, case, dtype, last):
    """One key's score of a row is +inf: inf - inf has no value, and the row is NaN. The
    other rows' score of that key is -inf: it has no part in them."""
    from magma_b200 import ops
    b, h, g, m, n, d = case
    q, k, v, do, _ = make(34, b, h, g, m, n, d, dtype)
    at = n - 1 if last else 0
    q[..., 0] = -1.0
    q[0, 0, m - 1, 0] = 1.0
    k[0, 0, at, 0] = math.inf
    keep = torch.arange(n, device="cuda") != at
    want, bound = reference(q[:1], k[:1, :, keep], v[:1, :, keep], do[:1], None, d ** -0.5)
    o, lse = ops.cross_attention_fwd(q, k, v)
    assert bool(torch.isnan(o[0, 0, m - 1]).all()) and math.isnan(lse[0, 0, m - 1].item())
    rows = slice(0, m - 1) if m > 1 else slice(0, 0)
    check(o[0, 0, rows], want[0][0, 0, rows], bound[0][0, 0, rows], "o")
    check(lse[0, 0, rows], want[1][0, 0, rows], bound[1][0, 0, rows], "lse")
    assert bool(torch.isfinite(o[b - 1, h - 1]).all()) and bool(torch.isfinite(lse[b - 1, h - 1]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", PATHS)
def test_a_row_of_scores_that_are_minus_infinity(cuda, case, dtype):
    """It comes out as a row without keys, on every path."""
    from magma_b200 import ops
    b, h, g, m, n, d = case
    q, k, v, do, _ = make(35, b, h, g, m, n, d, dtype)
    want, bound = reference(q, k, v, do, None, d ** -0.5)
    q[0, 0, m - 1] = 0.0
    q[0, 0, m - 1, 0] = 1.0
    k[0, 0, :, 0] = -math.inf
    o, lse = ops.cross_attention_fwd(q, k, v)
    assert bool((o[0, 0, m - 1] == 0).all()) and lse[0, 0, m - 1].item() == -math.inf
    if b * g == 1:  # all heads read these keys
        return
    check(o[b - 1, h - 1], want[0][b - 1, h - 1], bound[0][b - 1, h - 1], "o")
    check(lse[b - 1, h - 1], want[1][b - 1, h - 1], bound[1][b - 1, h - 1], "lse")
