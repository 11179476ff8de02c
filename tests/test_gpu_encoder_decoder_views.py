"""Outputs that lie between one another's positions, as the views of fused
projections do, are accepted and come out as those of their own memory do."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_cross_attention import make  # noqa: E402

pytestmark = pytest.mark.gpu


def views(kind, b, h, g, m, d, dtype):
    """q-, k- and v-shaped views of one buffer, in several layouts."""
    z = lambda *s: torch.full(s, 7.0, device="cuda", dtype=dtype)  # noqa: E731
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    if kind == "tokens":  # [B, S, (H + 2 G) D]
        x = z(b, m, h + 2 * g, d)
        return t(x[:, :, :h]), t(x[:, :, h:h + g]), t(x[:, :, h + g:])
    if kind == "heads":  # [B, H + 2 G, S, D]
        x = z(b, h + 2 * g, m, d)
        return x[:, :h], x[:, h:h + g], x[:, h + g:]
    if kind == "columns":  # [B, S, H, 3 D], the last heads unused in k and v
        x = z(b, m, h, 3 * d)
        return t(x[..., :d]), t(x[:, :, :g, d:2 * d]), t(x[:, :, :g, 2 * d:])
    # every third position of [B, H, 3 S, D]
    x = z(b, h, 3 * m, d)
    return x[:, :, ::3], x[:, :g, 1::3], x[:, :g, 2::3]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["tokens", "heads", "columns", "positions"])
@pytest.mark.parametrize("m", [1, 130])
def test_fused_gradients_and_inputs(cuda, kind, m, dtype):
    from magma_b200 import ops
    b, h, g, d = 2, 4, 2, 64
    q, k, v, do, _ = make(51, b, h, g, m, m, d, dtype)
    o, lse = ops.cross_attention_fwd(q, k, v)
    want = ops.cross_attention_bwd(q, k, v, o, do, lse)
    fused = views(kind, b, h, g, m, d, dtype)
    for x, y in zip(fused, (q, k, v)):
        x.copy_(y)
    out = views(kind, b, h, g, m, d, dtype)
    o2, lse2 = ops.cross_attention_fwd(*fused, out=out[0])
    assert torch.equal(lse, lse2) and torch.equal(o, o2)
    grads = views(kind, b, h, g, m, d, dtype)
    ops.cross_attention_bwd(*fused, o2, do, lse2, dq=grads[0], dk=grads[1], dv=grads[2])
    for x, y in zip(grads, want):
        assert torch.equal(x, y)


def test_an_output_beside_its_inputs(cuda):
    """The attention's output in the columns beside q, the table's gradient beside dout."""
    from magma_b200 import ops
    q, k, v, _, _ = make(52, 2, 4, 2, 70, 90, 64, torch.bfloat16)
    want, _ = ops.cross_attention_fwd(q, k, v)
    both = torch.zeros(2, 70, 4, 128, device="cuda", dtype=torch.bfloat16)
    both[..., :64] = q.transpose(1, 2)
    o = both[..., 64:].transpose(1, 2)
    ops.cross_attention_fwd(both[..., :64].transpose(1, 2), k, v, out=o)
    assert torch.equal(o, want) and torch.equal(both[..., :64].transpose(1, 2), q)
    tok = torch.randint(0, 20, (2, 10), device="cuda", dtype=torch.int32)
    wide = torch.randn(20, 40, device="cuda")
    want, _ = ops.embedding_scaled_bwd(tok, wide[:, :16].contiguous(), 20)
    ops.embedding_scaled_bwd(tok, wide[:, :16], 20, dtable=wide[:, 16:32])
    assert torch.equal(wide[:, 16:32], want)


def test_overlapping_views_are_refused(cuda):
    from magma_b200 import lib, ops
    x = torch.randn(2, 4, 80, 64, device="cuda")
    k = torch.randn(2, 2, 80, 64, device="cuda")
    q = x[:, :, :70]
    with pytest.raises(lib.MagmaError, match="memory"):
        ops.cross_attention_fwd(q, k, k, out=x[:, :, 1:71])
    o, lse = ops.cross_attention_fwd(q, k, k, out=x.new_empty(q.shape))
    pair = torch.empty(2, 2, 90, 64, device="cuda")
    with pytest.raises(lib.MagmaError, match="memory"):
        ops.cross_attention_bwd(q, k, k, o, o, lse, dk=pair[:, :, :80], dv=pair[:, :, 1:81])
    table = torch.randn(9, 64, device="cuda")
    tok = torch.zeros(1, 8, dtype=torch.int32, device="cuda")
    with pytest.raises(lib.MagmaError, match="memory"):
        ops.embedding_scaled_fwd(tok, table, out=table[1:])
    flat = torch.ones(10, device="cuda")
    with pytest.raises(lib.MagmaError, match="memory"):
        ops.clip_grad_norm([flat], 1.0, norm=flat[3:4])
