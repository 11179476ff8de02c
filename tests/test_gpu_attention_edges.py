"""Self-attention where the first keys of a row score -inf."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
def test_first_keys_score_minus_infinity(cuda, causal, dtype):
    """Rows from 128 on have the softmax of the other keys, whose scores are about -500.
    A score is off by u32 (D + 4) sum |q||k| / 8, 500 (D + 4) u32 = 2e-3, a probability by
    twice that; P and the output are rounded to their type (2^-8 in BF16)."""
    from magma_b200 import ops
    gen = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(2, 3, 400, 64, device="cuda", generator=gen).to(dtype) for _ in range(3))
    q[..., 0] = 1.0
    k[..., 0] = -4000.0
    k[:, :, :128, 0] = -math.inf
    o, lse = ops.attention_fwd(q, k, v, 0.125, causal)
    s = q.double() @ k.double().transpose(-1, -2) * 0.125
    if causal:
        s = s.masked_fill(torch.ones(400, 400, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    rows = slice(128, None) if causal else slice(None)
    s = s[:, :, rows]
    p = s.softmax(-1)
    want = p @ v.double()
    assert (lse[:, :, rows].double() - torch.logsumexp(s, -1)).abs().max() <= 2.5e-3
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    bound = (5e-3 + u) * (p @ v.double().abs()) + u * want.abs()
    assert bool(((o[:, :, rows].double() - want).abs() <= bound).all())
