"""Argument checks of the encoder-decoder operators (scaled embedding, cross
attention, gradient norm over many tensors), on a machine without a GPU: every
call here is refused before anything is launched, or has nothing to do."""
import ctypes as C

import pytest

from magma_b200 import lib

torch = pytest.importorskip("torch")

BUF = 0x100000  # an aligned address that a refused call never touches
OUT, OUT2, OUT3 = 0x10000000, 0x20000000, 0x30000000  # and others for outputs


def refused(name, *args):
    with pytest.raises(lib.MagmaError) as e:
        lib.call(name, *args)
    assert e.value.status == lib.INVALID_ARGUMENT
    return e.value.message


def st(*v):
    return (C.c_int64 * 3)(*v)


# ------------------------------------------------------------------- embedding
def emb_fwd(tokens=BUF, table=BUF, ld=8, pos=None, out=OUT, batch=2, seq=3, dim=8, vocab=5,
            ti=lib.F32, to=lib.F32):
    return ("magma_embedding_scaled_fwd", tokens, table, ld, pos, out, batch, seq, dim, vocab, 1.0,
            ti, to, None)


def emb_bwd(tokens=BUF, dout=BUF, dout_ld=8, dtable=OUT, dtable_ld=8, batch=2, seq=3, dim=8,
            vocab=5, pad=-1, ti=lib.F32, to=lib.F32, ws=BUF, ws_bytes=1 << 20):
    return ("magma_embedding_scaled_bwd", tokens, dout, dout_ld, dtable, dtable_ld, None, batch,
            seq, dim, vocab, 1.0, pad, 0, 0, ti, to, ws, ws_bytes, None)


@pytest.mark.parametrize("change,word", [
    (dict(batch=-1), "negative"), (dict(dim=1 << 23), "too large"), (dict(ti=lib.S32), "dtypes"),
    (dict(to=7), "dtypes"), (dict(tokens=None), "NULL"), (dict(table=None), "NULL"),
    (dict(out=None), "NULL"), (dict(ld=7), "table_ld"), (dict(vocab=0), "empty table"),
    (dict(batch=1 << 20, seq=1 << 20), "2^31"), (dict(out=BUF), "shares memory"),
])
def test_embedding_lookup_refuses(change, word):
    assert word in refused(*emb_fwd(**change))


@pytest.mark.parametrize("change,word", [
    (dict(seq=-1), "negative"), (dict(ti=lib.S64), "dtypes"), (dict(pad=5), "padding_idx"),
    (dict(pad=-2), "padding_idx"), (dict(dout=None), "NULL"), (dict(dtable=None), "NULL"),
    (dict(dout_ld=7), "dout_ld"), (dict(dtable_ld=0), "dtable_ld"), (dict(ws=None), "workspace"),
    (dict(ws_bytes=64), "workspace"), (dict(ws=BUF + 8), "workspace"), (dict(vocab=0), "empty"),
    (dict(dtable=BUF), "share memory"),
])
def test_embedding_gradient_refuses(change, word):
    assert word in refused(*emb_bwd(**change))


def test_embedding_without_rows_does_nothing():
    lib.call(*emb_fwd(tokens=None, table=None, out=None, batch=0))
    lib.call(*emb_bwd(tokens=None, dout=None, dtable=None, vocab=0, batch=0, ws=None))
    assert lib.query("magma_embedding_scaled_bwd_workspace_size", 0, 8, 8) == 0
    assert lib.query("magma_embedding_scaled_bwd_workspace_size", 4, 8, 8) >= 4 * 4 * 32


# ------------------------------------------------------------- cross attention
def fwd(q=BUF, k=BUF, v=BUF, o=OUT, batch=2, heads=4, kv_heads=2, m=3, n=5, hd=8, scale=1.0,
        dt=lib.F32, so=None, sq=None):
    sq = sq or st(heads * m * hd, m * hd, hd)
    sk = st(kv_heads * n * hd, n * hd, hd)
    return ("magma_cross_attention_fwd", q, k, v, o, None, None, batch, heads, kv_heads, m, n, hd,
            sq, sk, sk, so or st(heads * m * hd, m * hd, hd), scale, dt, None, 0, None)


def bwd(lse=BUF, dq=OUT, dk=OUT2, dv=OUT3, ws=BUF, ws_bytes=1 << 20, sdk=None, sdq=None, heads=4, kv_heads=2,
        m=3, n=5, hd=8, batch=2):
    sq = st(heads * m * hd, m * hd, hd)
    sk = st(kv_heads * n * hd, n * hd, hd)
    return ("magma_cross_attention_bwd", BUF, BUF, BUF, BUF, BUF, lse, None, dq, dk, dv, batch,
            heads, kv_heads, m, n, hd, sq, sk, sk, sq, sq, sdq or sq, sdk or sk, sk, 1.0, lib.F32,
            ws, ws_bytes, None)


@pytest.mark.parametrize("change,word", [
    (dict(batch=-1), "negative"), (dict(batch=1 << 16), "65536"), (dict(hd=129), "head_dim"),
    (dict(hd=0), "head_dim"), (dict(heads=5), "multiple"), (dict(dt=lib.S32), "dtype"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=-1.0), "scale"), (dict(q=None), "NULL"), (dict(k=None), "NULL"),
    (dict(v=None), "NULL"), (dict(o=None), "NULL"), (dict(sq=st(-1, 8, 8)), "stride"),
    (dict(so=st(96, 0, 8)), "share memory"), (dict(so=st(96, 24, 7)), "share memory"),
    (dict(so=st(8, 8, 8)), "share memory"), (dict(o=BUF), "shares memory"),
])
def test_cross_attention_refuses(change, word):
    assert word in refused(*fwd(**change))


@pytest.mark.parametrize("change,word", [
    (dict(lse=None), "NULL"), (dict(dq=None), "NULL"), (dict(dk=None), "NULL"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=16), "workspace"), (dict(ws=BUF + 4), "workspace"),
    (dict(sdk=st(80, 0, 8)), "share memory"), (dict(sdq=st(0, 24, 8)), "share memory"),
    (dict(dq=BUF), "shares memory"), (dict(dv=OUT2), "share memory"),
])
def test_cross_attention_gradient_refuses(change, word):
    assert word in refused(*bwd(**change))


def test_cross_attention_without_queries_does_nothing():
    lib.call(*fwd(q=None, k=None, v=None, o=None, batch=0))
    lib.call(*fwd(q=None, o=None, m=0))
    assert lib.query("magma_cross_attention_bwd_workspace_size", 0, 4, 2, 3, 5, 8, lib.F32) == 0


# ------------------------------------------------------------------------ clip
def clip(ptrs, outs, sizes, *, dts=None, odts=None, count=None, max_norm=1.0, norm=BUF, ws=BUF,
         ws_bytes=1 << 20):
    n = len(ptrs)
    arr = lambda t, v: (t * n)(*v)  # noqa: E731
    return ("magma_clip_grad_norm_multi", arr(C.c_void_p, ptrs), arr(C.c_void_p, outs),
            arr(C.c_int64, sizes), arr(C.c_int32, dts or [lib.F32] * n),
            arr(C.c_int32, odts or [lib.F32] * n), n if count is None else count, 1.0, max_norm,
            norm, ws, ws_bytes, None)


A, B_ = 0x200000, 0x300000


@pytest.mark.parametrize("args,kw,word", [
    (([A], [A], [4]), dict(count=-1), "negative count"),
    (([A], [A], [-4]), {}, "size"), (([None], [A], [4]), {}, "NULL tensor"),
    (([A], [None], [4]), {}, "NULL tensor"), (([A], [A], [4]), dict(dts=[3]), "F32 or BF16"),
    (([A], [A], [4]), dict(odts=[3]), "F32 or BF16"), (([A], [A], [4]), dict(max_norm=0.0), "max_norm"),
    (([A], [A], [4]), dict(max_norm=float("nan")), "max_norm"),
    (([A], [A], [4]), dict(norm=None), "norm"), (([A], [A], [4]), dict(ws=None), "workspace"),
    (([A], [A], [4]), dict(ws=BUF + 4), "workspace"), (([A + 2], [A + 2], [4]), {}, "aligned"),
    # the same tensor twice, partial overlaps, an output over another gradient,
    # in place with another dtype
    (([A, A], [A, A], [4, 4]), {}, "shares memory"),
    (([A, A + 8], [A, A + 8], [4, 4]), {}, "shares memory"),
    (([A, B_], [A, A], [4, 4]), {}, "shares memory"),
    (([A, B_], [B_, 0x400000], [4, 4]), {}, "shares memory"),
    (([A], [A + 4], [4]), {}, "shares memory"),
    (([A], [A], [4]), dict(odts=[lib.BF16]), "shares memory"),
])
def test_clip_refuses(args, kw, word):
    assert word in refused(*clip(*args, **kw))


def test_norm_workspace_grows_with_the_list():
    q = lambda n: lib.query("magma_grad_norm_multi_workspace_size", n)  # noqa: E731
    assert 0 < q(1) == q(1024) < q(1025)


# ---------------------------------------------------------------- torch front end
def test_front_end_refuses_host_tensors_and_wrong_lists():
    from magma_b200 import ops
    x = torch.zeros(2, 3, 4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.cross_attention_fwd(x, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.embedding_scaled_fwd(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(5, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.clip_grad_norm([torch.zeros(4)], 1.0)
    with pytest.raises(ValueError, match="at least one"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError, match="outputs for"):
        ops.clip_grad_norm([torch.zeros(4)], 1.0, out=[])
    with pytest.raises(ValueError, match="added to"):
        ops.embedding_scaled_bwd(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, 8), 5,
                                 accumulate=True)


# ---------------------------------------------------------- addresses off elements
@pytest.mark.parametrize("args", [
    fwd(q=BUF + 2), fwd(k=BUF + 1), fwd(v=BUF + 3), fwd(o=OUT + 2), fwd(q=BUF + 1, dt=lib.BF16),
    fwd(o=OUT + 1, dt=lib.BF16), bwd(lse=BUF + 2), bwd(dq=OUT + 2), bwd(dk=OUT2 + 1), bwd(dv=OUT3 + 2),
    emb_fwd(tokens=BUF + 2), emb_fwd(table=BUF + 2), emb_fwd(out=OUT + 1, to=lib.BF16),
    emb_fwd(pos=BUF + 2), emb_bwd(tokens=BUF + 1), emb_bwd(dout=BUF + 2),
    emb_bwd(dtable=OUT + 1, to=lib.BF16),
])
def test_addresses_off_their_elements_are_refused(args):
    assert "off its elements" in refused(*args)
