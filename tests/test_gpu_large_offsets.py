"""Tensors of more than 2^31 elements: offsets past 32 bits in the embedding, the log probabilities and the gradient norm.  Rows at
both ends are checked against the same rows by themselves."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_embedding_table():
    from hawk_b200 import embedding, ops
    V, H = (1 << 31) // 1024 + 77, 1032   # 2.24e9 elements
    w = torch.empty(V, H, dtype=BF16, device="cuda")
    ids = torch.tensor([0, V - 1, V // 2, V - 1, 5], device="cuda")
    w[ids] = torch.randn(5, H, device="cuda").to(BF16)
    assert torch.equal(embedding(ids, w), w[ids])
    del w
    go = torch.randn(5, H, device="cuda").to(BF16)
    dw = ops.embedding_bwd(ids, go, V, 1.0, -1)
    assert torch.equal(dw[V - 1], (go[1].float() + go[3].float()).to(BF16)) and torch.equal(dw[V // 2], go[2])
    assert int((dw.view(-1).view(torch.int16).view(V, H) != 0).any(1).sum()) == 4


def test_embedded_tokens():
    from hawk_b200 import embedding, ops
    N, H = (1 << 31) // 2048 + 1000, 2048
    w = torch.randn(50, H, device="cuda").to(BF16)
    ids = torch.arange(N, device="cuda") % 50
    out = embedding(ids, w)
    assert torch.equal(out[-3:], w[ids[-3:]]) and torch.equal(out[:3], w[:3])
    out.zero_()
    out[-1], out[0] = 1.0, 2.0
    dw = ops.embedding_bwd(ids, out, 50, 1.0, -1)
    last = int(ids[-1])
    assert float(dw[last, 7]) == 1.0 and float(dw[0, 2047]) == 2.0 and float(dw.float().sum()) == 3.0 * H


def test_logits():
    from hawk_b200 import token_logprobs
    N, V = (1 << 31) // 32000 + 500, 32000
    x = torch.zeros(N, V, dtype=BF16, device="cuda")
    ends = torch.tensor([0, 1, N - 2, N - 1], device="cuda")
    x[ends] = (3 * torch.randn(4, V, device="cuda")).to(BF16)
    t = torch.arange(N, device="cuda") % V
    x = x.requires_grad_()
    lp, H, best, ids = token_logprobs(x, t, 3)
    small = x.detach()[ends].requires_grad_()
    want = token_logprobs(small, t[ends], 3)
    # four rows are cut over more blocks, so their sums are in another order: each is within 8e-6 + 2^-22 |log p| of the exact one
    # (3e-5 (1 + H) the entropy), and 2^-8 |d x| covers a bf16 rounding that falls on the other side
    for a, b in zip((lp, best, H), (want[0], want[2], want[1])):
        assert float((a[ends] - b).abs().max()) <= (7e-4 if a is H else 3e-5)
    assert torch.equal(ids[ends], want[3])
    up = torch.randn(N, device="cuda")
    dx, = torch.autograd.grad((lp, H), x, (up, up))
    ds, = torch.autograd.grad(want[:2], small, (up[ends], up[ends]))
    assert bool(((dx[ends].float() - ds.float()).abs() <= 2.0 ** -7 * ds.float().abs() + 1e-6).all())


def test_linear_logprobs():
    from hawk_b200 import linear_logprobs
    N, V, H = (1 << 31) // 32000 + 500, 32000, 64
    w = torch.randn(V, H, device="cuda").to(BF16)
    a = torch.randn(N, H, device="cuda").to(BF16)
    t = torch.randint(0, V, (N,), device="cuda")
    t[2000:-2000] = -1
    ends = torch.cat([torch.arange(2000), torch.arange(N - 2000, N)]).cuda()
    up = torch.randn(N, device="cuda") / 4000
    aa, ab, wa, wb = (z.detach().requires_grad_() for z in (a, a[ends], w, w))
    full, part = linear_logprobs(wa, aa, t), linear_logprobs(wb, ab, t[ends])
    assert all(torch.equal(x[ends], y) for x, y in zip(full, part))
    g = torch.autograd.grad(full, (wa, aa), (up, up))
    h = torch.autograd.grad(part, (wb, ab), (up[ends], up[ends]))
    # the sums over the vocabulary may be cut differently, and those over the rows are: bf16 results of the same fp32 sums
    assert float((g[1][ends].float() - h[1].float()).norm() / h[1].float().norm()) <= 4e-3
    assert float((g[0].float() - h[0].float()).norm() / h[0].float().norm()) <= 4e-3
    assert float(g[1][2000:-2000].abs().max()) == 0


def test_norm():
    from hawk_b200 import grad_norm
    t = torch.zeros((1 << 31) + 12345, dtype=BF16, device="cuda")
    t[0], t[-1], t[1 << 31] = 3.0, 4.0, 12.0
    assert float(grad_norm([t])) == 13.0
