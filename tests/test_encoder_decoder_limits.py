"""Limits of the encoder-decoder operators' arguments, on a machine without a GPU."""
import pytest

from magma_b200 import lib

pytest.importorskip("torch")

from test_encoder_decoder_refusals import bwd, fwd, refused  # noqa: E402


@pytest.mark.parametrize("args", [fwd(m=(1 << 31) - 63), fwd(n=(1 << 31) - 1), bwd(m=(1 << 31) - 1),
                                  bwd(n=(1 << 31) - 63), fwd(m=1 << 31)])
def test_lengths_whose_padding_would_not_fit_32_bits_are_refused(args):
    assert "2^31 - 64" in refused(*args)


def test_workspace_queries_beyond_the_limit_ask_for_nothing_to_launch():
    for n in ((1 << 31) - 63, 1 << 31):
        assert lib.query("magma_cross_attention_fwd_workspace_size", 1, 1, 1, n, 8, 8, lib.BF16) == 0


def test_a_norm_off_its_element_is_refused():
    """Its store would fault."""
    from test_encoder_decoder_refusals import BUF, OUT, clip
    assert "norm" in refused(*clip([OUT], [OUT], [4], norm=BUF + 2))
    name, grads, _, sizes, dtypes, *_ = clip([OUT], [OUT], [4])
    assert "norm" in refused("magma_grad_norm_multi", grads, sizes, dtypes, 1, 1.0, BUF + 1, OUT, 1 << 20, None)
