"""The encoder-decoder operators together: one training step of a cross-attention
block (embedding, projections, attention over a padded source, its gradients,
clipping, Adam) and a decoding step after it, as a program would run them.

Tolerance of the gradients: eight F32 products follow one another, each at most
K u off relative to the product of its operands' sizes (K = 96 terms, u = 2^-24),
which for operands without a sign pattern is sqrt(K) times the size of the
product: 8 * 96 * 2^-24 * sqrt(96) = 4.5e-4 in norm.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TOL = 8 * 96 * 2.0 ** -24 * math.sqrt(96)
B, M, N, D, H, G, V, PAD = 3, 37, 70, 96, 4, 2, 50, 0
HD = D // H


def parameters(seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return {"table": r(V, D) / D ** 0.5, "pos": 0.1 * r(M, D), "wq": r(D, D) / D ** 0.5,
            "wkv": r(2 * G * HD, D) / D ** 0.5, "wo": r(D, D) / D ** 0.5}


def batch(seed=1):
    g = torch.Generator("cuda").manual_seed(seed)
    src = torch.randint(1, V, (B, N), device="cuda", generator=g).int()
    tgt = torch.randint(1, V, (B, M), device="cuda", generator=g).int()
    lens = torch.tensor([N, 41, 0], dtype=torch.int32, device="cuda")
    src[torch.arange(N, device="cuda")[None] >= lens[:, None]] = PAD
    return src, tgt, lens, torch.randn(B * M, D, device="cuda", generator=g)


def step(ops, p, src, tgt, lens, dy):
    """Loss sum(y dy) and the gradients of every parameter, from library calls."""
    scale = D ** 0.5
    xs = ops.embedding_scaled_fwd(src, p["table"], scale=scale)
    xt = ops.embedding_scaled_fwd(tgt, p["table"], p["pos"], scale=scale)
    q = ops.gemm(xt, p["wq"], trans_b=True).view(B, M, H, HD).transpose(1, 2)
    kv = ops.gemm(xs, p["wkv"], trans_b=True).view(B, N, 2, G, HD)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    o, lse = ops.cross_attention_fwd(q, k, v, kv_lens=lens)
    ot = o.transpose(1, 2).reshape(B * M, D)
    y = ops.gemm(ot, p["wo"], trans_b=True)
    g = {"wo": ops.gemm(dy, ot, trans_a=True)}
    do = ops.gemm(dy, p["wo"]).view(B, M, H, HD).transpose(1, 2)
    dkv = torch.empty_like(kv)  # the gradient of the fused projection, written in place
    dq, _, _ = ops.cross_attention_bwd(q, k, v, o, do, lse, kv_lens=lens,
                                       dk=dkv[:, :, 0].transpose(1, 2),
                                       dv=dkv[:, :, 1].transpose(1, 2))
    dq, dkv = dq.transpose(1, 2).reshape(B * M, D), dkv.view(B * N, -1)
    g["wq"] = ops.gemm(dq, xt, trans_a=True)
    g["wkv"] = ops.gemm(dkv, xs, trans_a=True)
    g["table"], _ = ops.embedding_scaled_bwd(src, ops.gemm(dkv, p["wkv"]), V, scale=scale,
                                             padding_idx=PAD)
    _, g["pos"] = ops.embedding_scaled_bwd(tgt, ops.gemm(dq, p["wq"]), V, scale=scale,
                                           padding_idx=PAD, pos=True, dtable=g["table"],
                                           accumulate=True)
    return y, g, (q, k, v, o)


def definition(p, src, tgt, lens, dy):
    p = {n: t.double().requires_grad_() for n, t in p.items()}
    emb = lambda t: torch.nn.functional.embedding(t.long(), p["table"], padding_idx=PAD)  # noqa: E731
    xs, xt = emb(src) * D ** 0.5, emb(tgt) * D ** 0.5 + p["pos"]
    q = (xt @ p["wq"].T).view(B, M, H, HD).transpose(1, 2)
    kv = (xs @ p["wkv"].T).view(B, N, 2, G, HD)
    k, v = (kv[:, :, i].transpose(1, 2).repeat_interleave(H // G, 1) for i in (0, 1))
    mask = (torch.arange(N, device="cuda")[None] < lens[:, None])[:, None, None, :]
    s = (q @ k.transpose(-1, -2) * HD ** -0.5).masked_fill(~mask, -1e300)
    o = torch.where(mask.any(-1, keepdim=True), torch.softmax(s, -1) @ v, 0.0)
    y = o.transpose(1, 2).reshape(B * M, D) @ p["wo"].T
    (y * dy.double()).sum().backward()
    return y.detach(), {n: t.grad for n, t in p.items()}


def off(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def test_training_step(cuda):
    from magma_b200 import ops
    p, data = parameters(), batch()
    y, g, _ = step(ops, p, *data)
    wy, wg = definition(p, *data)
    assert off(y, wy) <= TOL
    for n in g:
        assert off(g[n], wg[n]) <= TOL, n
    assert bool((g["table"][PAD] == 0).all())
    # clipping and Adam over the separate tensors, against the same in 64 bits
    names = sorted(g)
    norm = ops.clip_grad_norm([g[n] for n in names], 1.0)
    want = math.sqrt(sum(float(wg[n].square().sum()) for n in names))
    assert abs(norm.item() - want) <= TOL * want
    for n in names:
        assert off(g[n], wg[n] / want) <= 2 * TOL
    before = {n: p[n].clone() for n in names}
    zeros = lambda: [torch.zeros_like(p[n]) for n in names]  # noqa: E731
    ops.adam_step_multi([p[n] for n in names], [g[n] for n in names], zeros(), zeros(), step=1, lr=1e-3)
    for n in names:
        moved = (p[n] - before[n])[g[n].abs() > 1e-6]
        assert bool((moved.abs() <= 1.01e-3).all()) and bool((moved.abs() > 0).all())
    assert ops.device_error_check() == 0


def test_training_step_in_a_graph_is_the_eager_one(cuda):
    from magma_b200 import ops
    p, data = parameters(), batch()
    y, g, _ = step(ops, p, *data)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            y2, g2, _ = step(ops, p, *data)
        for _ in range(2):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y2)
    for n in g:
        assert torch.equal(g[n], g2[n]), n


def test_decoding_step_is_the_last_row(cuda):
    """One query per sequence gives the last row of the whole pass: both are off the
    definition by a row's error at most (D + n terms of 2^-24 of the values' size)."""
    from magma_b200 import ops
    p, data = parameters(), batch()
    _, _, (q, k, v, o) = step(ops, p, *data)
    lens = data[2]
    one, _ = ops.cross_attention_fwd(q[:, :, -1:], k, v, kv_lens=lens)
    bound = 2 * (4 * HD + 2 * N + 64) * 2.0 ** -24 * v.abs().max().item() * max(
        1.0, q.abs().max().item() * k.abs().max().item())
    assert (one - o[:, :, -1:]).abs().max().item() <= bound
    assert bool((one[2] == 0).all())
