"""Outputs that share memory with another tensor of their call, without a GPU: every
call here is refused before anything is launched."""
import ctypes as C

import pytest

from magma_b200 import lib

pytest.importorskip("torch")

from test_encoder_decoder_refusals import (BUF, OUT, OUT2, OUT3, clip, emb_bwd, emb_fwd,  # noqa: E402
                                           refused, st)

Q, K, V, O, DO, LSE, LENS = (0x40000000 + i * 0x1000000 for i in range(7))
ROW = 32  # bytes of a position of eight F32 values


def fwd(q=Q, k=K, v=V, o=OUT, lse=LSE, lens=LENS, sq=None, so=None):
    """Two sequences of four heads over two, three queries, five keys."""
    sq, sk = sq or st(96, 24, 8), st(80, 40, 8)
    return ("magma_cross_attention_fwd", q, k, v, o, lse, lens, 2, 4, 2, 3, 5, 8, sq, sk, sk,
            so or st(96, 24, 8), 1.0, lib.F32, None, 0, None)


def bwd(lse=LSE, lens=LENS, dq=OUT, dk=OUT2, dv=OUT3, sdk=None, sdv=None):
    sq, sk = st(96, 24, 8), st(80, 40, 8)
    return ("magma_cross_attention_bwd", Q, K, V, O, DO, lse, lens, dq, dk, dv, 2, 4, 2, 3, 5, 8, sq,
            sk, sk, sq, sq, sq, sdk or sk, sdv or sk, 1.0, lib.F32, BUF, 1 << 20, None)


@pytest.mark.parametrize("args", [
    # a row into an input, over its last row, its first row behind the output's last
    fwd(o=Q + ROW), fwd(o=Q + 23 * ROW), fwd(o=Q - 23 * ROW), fwd(o=K + 19 * ROW), fwd(o=V + ROW),
    fwd(o=Q + 4), fwd(o=LENS + 4), fwd(o=LENS - 23 * ROW), fwd(lse=Q + 8), fwd(lse=K + 4), fwd(lse=OUT),
    fwd(lse=OUT - 4 * 23), fwd(lse=LENS), fwd(lse=LENS + 4),
    # the output's positions in the gaps of a wider q, and one element too far
    fwd(sq=st(192, 48, 16), so=st(192, 48, 16), o=Q + 28),
    # a broadcast q inside the output
    fwd(q=OUT + 23 * ROW, sq=st(0, 0, 0)),
])
def test_cross_attention_outputs_over_inputs(args):
    assert "memory" in refused(*args)


@pytest.mark.parametrize("args", [
    bwd(dq=Q + ROW), bwd(dq=DO + ROW), bwd(dq=O - 4), bwd(dk=K + 4), bwd(dv=K - 4), bwd(dq=LSE + 4),
    bwd(dk=LENS), bwd(dv=LENS + 4), bwd(dk=OUT3 + ROW), bwd(dv=OUT2 - 19 * ROW), bwd(dk=OUT + ROW),
    # dk and dv of a fused buffer, one element too close
    bwd(dk=OUT2, dv=OUT2 + 60, sdk=st(160, 16, 32), sdv=st(160, 16, 32)),
])
def test_cross_attention_gradients_over_other_tensors(args):
    assert "memory" in refused(*args)


@pytest.mark.parametrize("args", [
    emb_fwd(out=BUF + 4, tokens=Q), emb_fwd(out=BUF - 5 * ROW, tokens=Q), emb_fwd(out=Q + 20, tokens=Q),
    emb_fwd(out=V + ROW, pos=V), emb_fwd(out=BUF + 28, tokens=Q, ld=16),
    emb_bwd(dtable=BUF + ROW, tokens=Q, ws=K), emb_bwd(dtable=BUF - 4 * ROW, tokens=Q, ws=K),
    emb_bwd(dtable=Q + 20, tokens=Q, ws=K), emb_bwd(dtable=BUF + 28, tokens=Q, ws=K, dout_ld=16, dtable_ld=16),
])
def test_embedding_outputs_over_inputs(args):
    assert "memory" in refused(*args)


@pytest.mark.parametrize("dpos", [OUT, OUT + 4 * ROW, OUT - 2 * ROW, BUF + ROW, Q + 4])
def test_position_gradient_over_other_tensors(dpos):
    args = list(emb_bwd(tokens=Q, ws=K))
    args[6] = dpos
    assert "memory" in refused(*args)


@pytest.mark.parametrize("norm", [OUT, OUT + 12, OUT2 + 4])
def test_norm_inside_a_clipped_tensor(norm):
    assert "shares memory" in refused(*clip([OUT, OUT2], [OUT, OUT3], [4, 4], norm=norm))
