"""An error that one call reports is not reported again by the next."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_a_failed_call_leaves_no_error_for_the_next(cuda):
    from magma_b200 import lib, ops
    tok = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    table = torch.randn(3, 16, device="cuda")
    q = torch.randn(1, 2, 100, 64, device="cuda")
    want, _ = ops.cross_attention_fwd(q, q, q)
    p = C.c_void_p()
    for call in (lambda: ops.embedding_scaled_fwd(tok, table), lambda: ops.cross_attention_fwd(q, q, q)[0],
                 lambda: ops.embedding_scaled_bwd(tok, table[:1].repeat(4, 1), 3)[0]):
        before = call()
        with pytest.raises(lib.MagmaError):
            lib.call("magma_malloc", C.byref(p), 1 << 60)  # more than any device has
        assert torch.equal(call(), before)
