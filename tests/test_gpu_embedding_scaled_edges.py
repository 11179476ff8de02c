"""The scaled embedding's gradient at its widest rows."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_embedding_scaled import UNIT, check, gradient_reference  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("td,tt", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("d", [2097153, 1 << 22])
@pytest.mark.parametrize("accumulate", [False, True])
def test_rows_of_more_columns_than_a_grid_has_blocks(cuda, d, td, tt, accumulate):
    """A run of equal tokens that crosses the shares of 8 places, in rows whose 32-column
    blocks outnumber a grid's second dimension (65535); odd widths and shifted rows are
    added up by single columns."""
    from magma_b200 import ops
    tok = torch.zeros(1, 17, dtype=torch.int32, device="cuda")
    tok[0, 3] = 1
    gen = torch.Generator("cuda").manual_seed(41)
    wide = torch.randn(17, d + 1, device="cuda", generator=gen).to(td)
    dout = wide[:, 1:]
    old = torch.randn(2, d, device="cuda", generator=gen).to(tt) if accumulate else None
    dtable = old.clone() if accumulate else None
    got, dpos = ops.embedding_scaled_bwd(tok, dout, 2, scale=1.5, pos=True, dtype=tt,
                                         dtable=dtable, accumulate=accumulate)
    want, bound = gradient_reference(tok, dout, 2, 1.5, None, old)
    check(got, want, bound + UNIT[tt] * want.abs(), "dtable")
    assert torch.equal(dpos, dout.float())
    assert ops.device_error_check() == 0
