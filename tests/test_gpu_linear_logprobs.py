"""Log probabilities and entropies from activations and head weight, and both gradients, against plain ones in 64 bits on the
bf16 operands.

Tolerances.  A logit is an fp32 sum of H exact products: off by less than H 2^-24 sum |a w| (measured far less: pairwise inside the
tensor core); with |a||w| <= 8 sqrt(H) here and errors that do not conspire, 2^-20 of the logits' spread; log s adds 8e-6 as in
the logits' own test: 3e-5 absolute in a log probability, 1e-4 in the entropy.  Gradients: d x is e rounded to fp16 (2^-12, or
2^-25 of its group's largest) times factors right to 1e-4, rounded to bf16 (2^-8 half a step of eps 2^-7): 2^-8 + 4e-4 per element
and, over sums of many, norm-wise; the result rounds once more (2^-8 in bf16).  Independent roundings of at most 2^-8 relative have
a root mean square of 2^-8 / sqrt(3) or less: sqrt(2) of that, 3.2e-3; 6e-3 leaves room for few terms."""
import math

import pytest
import torch

from conftest import rel_l2

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _case(N, H, V, seed=0, dtype=BF16, w_dtype=None, lift=16.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, H, generator=g, device="cuda") / math.sqrt(H)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    a = torch.randn(N, H, generator=g, device="cuda") + w[t] * (lift * torch.rand(N, 1, generator=g, device="cuda"))
    t[0] = 0
    t[-1] = V - 1
    gl, ge = torch.randn(N, generator=g, device="cuda"), torch.randn(N, generator=g, device="cuda") * 0.3
    return w.bfloat16().to(w_dtype or dtype), a.bfloat16().to(dtype), t, gl, ge


def _reference(w, a, t, gl, ge):
    """(lp, H, dw, da) in 64 bits, rows in pieces."""
    out = []
    dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    for r in range(0, t.numel(), 4096):
        ar, tr, glr, ger = a[r:r + 4096].double(), t[r:r + 4096], gl[r:r + 4096].double(), ge[r:r + 4096].double()
        named = tr >= 0
        ar = torch.where(named[:, None], ar, 0)
        logp = torch.log_softmax(ar @ w.double().T, -1)
        p = logp.exp()
        H = -(p * logp).sum(-1)
        at = tr.clamp(0, w.shape[0] - 1)[:, None]
        d = -p * (glr[:, None] + ger[:, None] * (logp + H[:, None]))
        d.scatter_add_(1, at, glr[:, None])
        d = torch.where(named[:, None], d, 0)
        dw += d.T @ ar
        out.append((torch.where(named, logp.gather(1, at)[:, 0], 0), torch.where(named, H, 0), d @ w.double()))
    lp, H, da = (torch.cat(x) for x in zip(*out))
    return lp, H, dw, da


def _check(w, a, t, gl, ge, tol=6e-3):
    from hawk_b200 import check_device_status, linear_logprobs
    w, a = w.detach().requires_grad_(), a.detach().requires_grad_()
    lp, H = linear_logprobs(w, a, t)
    dw, da = torch.autograd.grad((lp, H), (w, a), (gl, ge))
    with torch.no_grad():
        lp0, H0 = linear_logprobs(w, a, t)
    check_device_status()
    assert lp.dtype == H.dtype == F32 and dw.dtype == w.dtype and da.dtype == a.dtype
    assert torch.equal(lp, lp0) and torch.equal(H, H0)  # with and without what a backward needs
    rlp, rH, rdw, rda = _reference(w.detach(), a.detach(), t, gl, ge)
    named = t >= 0
    spread = float((a.detach().double()[named] @ w.detach().double().T).abs().max()) * 2.0 ** -20  # of the logits
    assert float((lp - rlp).abs().max()) <= 3e-5 + spread and float((H - rH).abs().max()) <= 1e-4 + spread
    assert rel_l2(dw, rdw) <= tol and rel_l2(da, rda) <= tol
    return lp, H, dw, da


@pytest.mark.parametrize("N,H,V", [(1, 8, 1), (1, 8, 2), (2, 64, 127), (5, 72, 128), (1, 2048, 32000), (33, 64, 129), (255, 128, 257), (256, 64, 1000),
                                   (257, 512, 383), (1548, 512, 32000), (700, 1000, 4097), (2100, 32, 97), (4096, 2048, 2048)])
def test_values_and_gradients(N, H, V):
    _check(*_case(N, H, V, N + H + V))


@pytest.mark.parametrize("dtype,w_dtype", [(F32, F32), (BF16, F32), (F32, BF16)])
def test_operand_types(dtype, w_dtype):
    w, a, t, gl, ge = _case(300, 128, 1003, 5, dtype, w_dtype)
    got = _check(w, a, t, gl, ge)
    same = _check(w.bfloat16(), a.bfloat16(), t, gl, ge)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
    assert torch.equal(got[2].bfloat16(), same[2]) and torch.equal(got[3].bfloat16(), same[3])


def test_one_gradient_only():
    from hawk_b200 import linear_logprobs
    w, a, t, gl, ge = _case(200, 64, 500, 6)
    both = _check(w, a, t, gl, ge)
    for k in (0, 1):
        ops = [w.detach(), a.detach()]
        ops[k].requires_grad_()
        lp, H = linear_logprobs(*ops, t)
        g, = torch.autograd.grad((lp, H), (ops[k],), (gl, ge))
        assert torch.equal(g, both[2 + k])
        for out, up, zero in ((0, gl, ge), (1, ge, gl)):  # one of the two results used
            res = linear_logprobs(*ops, t)
            g, = torch.autograd.grad(res[out], (ops[k],), up)
            ref = _reference(w, a, t, gl if out == 0 else gl * 0, ge if out == 1 else ge * 0)
            assert rel_l2(g, ref[2 + k]) <= 6e-3


def test_backward_twice():
    from hawk_b200 import linear_logprobs
    w, a, t, gl, ge = _case(130, 64, 300, 7)
    w, a = w.requires_grad_(), a.requires_grad_()
    out = linear_logprobs(w, a, t)
    one = torch.autograd.grad(out, (w, a), (gl, ge), retain_graph=True)
    two = torch.autograd.grad(out, (w, a), (gl, ge))
    assert all(torch.equal(x, y) for x, y in zip(one, two))


@pytest.mark.parametrize("share", [0.2, 1.0])
def test_left_out_rows_hold_anything(share):
    from hawk_b200 import linear_logprobs
    w, a, t, gl, ge = _case(400, 64, 777, 8)
    g = torch.Generator(device="cuda").manual_seed(1)
    t = torch.where(torch.rand(400, generator=g, device="cuda") < share, -1 - t, t)
    clean = _check(w, a, t, gl, ge) if share < 1 else None
    out = t < 0
    a = torch.where(out[:, None], torch.tensor([math.nan, math.inf], device="cuda", dtype=BF16)[torch.arange(400, device="cuda") % 2][:, None], a)
    w, a = w.requires_grad_(), a.requires_grad_()
    lp, H = linear_logprobs(w, a, t)
    dw, da = torch.autograd.grad((lp, H), (w, a), (gl, ge))
    assert float(lp[out].abs().max()) == 0 and float(H[out].abs().max()) == 0 and float(da[out].abs().max()) == 0
    if clean is None:
        assert float(dw.abs().max()) == 0
    else:
        assert torch.equal(lp, clean[0]) and torch.equal(H, clean[1]) and torch.equal(dw, clean[2]) and torch.equal(da, clean[3])


def test_certain_and_huge_logits():
    """Tokens that are all but certain, where 1 - p and log p are what is left of large numbers."""
    w, a, t, gl, ge = _case(256, 256, 1000, 9, lift=60.0)
    lp, H, dw, da = _check(w, a, t, gl, ge, tol=1e-2)
    assert float(lp.max()) > -1e-6
    # a row's gradient by itself, where p is near 1: against its own size, not the batch's
    from hawk_b200 import linear_logprobs
    rlp, rH, _, rda = _reference(w, a, t, gl, ge * 0)
    a = a.detach().requires_grad_()
    one, = torch.autograd.grad(linear_logprobs(w, a, t)[0], a, gl)
    sure = (rlp > -0.05) & (rlp < -1e-4)
    err = (one.double() - rda).norm(dim=1) / rda.norm(dim=1)
    assert int(sure.sum()) > 3 and float(err[sure].max()) <= 1.2e-2  # 2^-8 + 2^-9 of d x per element, and 1 - p right to 1e-5 / 1e-4 absolute
    big = w.detach() * 30
    _check(big, a.detach(), t, gl, ge * 0, tol=1e-2)


def test_shapes_strides_and_tokens():
    from hawk_b200 import linear_logprobs
    w, a, t, gl, ge = _case(24, 64, 301, 10)
    lp, H = linear_logprobs(w, a, t)
    assert all(torch.equal(x, y.view(4, 6)) for x, y in zip(linear_logprobs(w, a.view(4, 6, 64), t.view(4, 6)), (lp, H)))
    wide = torch.zeros(24, 130, dtype=BF16, device="cuda")
    wide[:, 1:65] = a
    assert all(torch.equal(x, y) for x, y in zip(linear_logprobs(w.t().contiguous().t(), wide[:, 1:65], t.int()), (lp, H)))
    one = linear_logprobs(w, a[3], t[3])
    assert one[0].shape == () and float(one[0]) == float(lp[3])
    bad = t.clone()
    bad[5], bad[6] = 301, 2 ** 40
    x = a.detach().requires_grad_()
    lp2, H2 = linear_logprobs(w, x, bad)
    assert bool(lp2[5:7].isnan().all()) and torch.equal(H2, H) and torch.equal(lp2[7:], lp[7:])
    dx, = torch.autograd.grad(lp2, x, gl)
    assert bool(dx[5:7].isnan().all()) and bool(dx[7:].isfinite().all())
    e = linear_logprobs(w.requires_grad_(), a[:0], t[:0])
    dw, = torch.autograd.grad(e[0].sum(), w)
    assert e[0].shape == (0,) and float(dw.abs().max()) == 0


def test_agrees_with_the_mean_loss():
    """The mean cross-entropy over the same rows, whose logits are rounded to bf16: 2^-9 of logits up to 20, averaged."""
    from hawk_b200 import fused_cross_entropy, linear_logprobs
    w, a, t, *_ = _case(600, 128, 1000, 11)
    assert abs(float(-linear_logprobs(w, a, t)[0].mean()) - float(fused_cross_entropy(w, a, t))) <= 1e-2


def test_refusals():
    from hawk_b200 import linear_logprobs
    w, a, t, *_ = _case(6, 64, 50, 12)
    with pytest.raises(ValueError, match="weight of shape"):
        linear_logprobs(w, a[:, :32], t)
    with pytest.raises(ValueError, match="tokens of shape"):
        linear_logprobs(w, a, t[:3])
    with pytest.raises(TypeError, match="integers"):
        linear_logprobs(w, a, t.float())
    with pytest.raises(TypeError, match="float16"):
        linear_logprobs(w, a.half(), t)
    with pytest.raises(RuntimeError, match="multiple"):
        linear_logprobs(w[:, :12], a[:, :12], t)
    with pytest.raises(RuntimeError, match="cpu"):
        linear_logprobs(w, a, t.cpu())


def test_captured_forward_and_backward():
    from hawk_b200 import ops
    w, a, t, gl, ge = _case(150, 64, 400, 13)

    def both():
        lp, H, saved = ops.linear_logprobs_fwd(w, a, t, True)
        return (lp, H, *ops.linear_logprobs_bwd(w, a, t, saved, lp, H, gl, ge, True, True))
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    w2, a2, t2, gl2, ge2 = _case(150, 64, 400, 14)
    for x, y in ((w, w2), (a, a2), (t, t2), (gl, gl2), (ge, ge2)):
        x.copy_(y)
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(out, both()))


@pytest.mark.parametrize("N,H,V", [(600, 64, 777), (70, 32, 300), (20000, 32, 97), (5000, 512, 1000)])
def test_any_number_of_named_rows(N, H, V):
    """The products run over the rows that name a token alone: counts at the edges of their tiles, blocks and splits of K, in scattered
    places, and NaN where a row is left out."""
    w, a, t, gl, ge = _case(N, H, V, N)
    g = torch.Generator(device="cuda").manual_seed(3)
    for count in sorted({0, 1, 2, 63, 64, 65, 255, 256, 257, N // 2, N - 1, N}):
        if count > N:
            continue
        keep = torch.randperm(N, generator=g, device="cuda")[:count]
        some = torch.full_like(t, -1)
        some[keep] = t[keep]
        rows = torch.full_like(a, math.nan)
        rows[keep] = a[keep]
        if count:
            lp, H_, dw, da = _check(w, rows, some, gl, ge)
        else:
            from hawk_b200 import linear_logprobs
            x, y = w.detach().requires_grad_(), rows.requires_grad_()
            lp, H_ = linear_logprobs(x, y, some)
            dw, da = torch.autograd.grad((lp, H_), (x, y), (gl, ge))
            assert float(dw.abs().max()) == 0
        out = some < 0
        assert all(bool((x[out] == 0).all()) for x in (lp, H_, da))


def test_replays_with_other_masks():
    from hawk_b200 import ops
    w, a, t, gl, ge = _case(300, 64, 400, 15)

    def both():
        lp, H, saved = ops.linear_logprobs_fwd(w, a, t, True)
        return (lp, H, *ops.linear_logprobs_bwd(w, a, t, saved, lp, H, gl, ge, True, True))
    both()
    torch.cuda.synchronize()
    full, graph = t.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for share in (0.0, 0.1, 0.9, 1.0, 0.5):
        t.copy_(torch.where(torch.arange(300, device="cuda") * 7 % 300 < share * 300, -1, full))
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(out, both()))


@pytest.mark.parametrize("N", [32768, 32769, 100003])
@pytest.mark.parametrize("share", [0.0, 0.3])
def test_long_lists_of_rows(N, share):
    """Lists on both sides of where their blocks are counted first, and the number of launches that goes with it."""
    from hawk_b200 import ops
    w, a, t, gl, ge = _case(N, 32, 70, 16)
    g = torch.Generator(device="cuda").manual_seed(2)
    t = torch.where(torch.rand(N, generator=g, device="cuda") < share, -3, t)
    ops.LOG.reset()
    _check(w, a, t, gl, ge)
    counts = dict(ops.LOG.counts)
    ops.LOG.enabled = False
    assert counts["linear_logprobs"] == 2 * (4 if N > 32768 else 3)


@pytest.mark.parametrize("N,H,V,lift", [(31, 96, 5802, 1.0), (64, 512, 4000, 16.0), (1000, 128, 4000, 16.0)])
def test_activations_gradient_is_rounded_once(N, H, V, lift):
    """The token's element of d x, most of a row where the other probabilities are small, is held exactly: what is left is the
    result's own rounding, in norm within a tenth of that of the 64-bit gradient, and 2^-8 of the other elements' part."""
    from hawk_b200 import linear_logprobs
    for seed in range(4):
        w, a, t, gl, ge = _case(N, H, V, seed, lift=lift)
        _, _, _, da = _reference(w, a, t, gl, ge)
        a.requires_grad_()
        got, = torch.autograd.grad(linear_logprobs(w, a, t), a, (gl, ge))
        assert rel_l2(got, da) <= 1.1 * rel_l2(da.bfloat16(), da)


@pytest.mark.parametrize("N", [1, 31, 64, 65, 128])
def test_weights_gradient_of_few_rows_is_rounded_once(N):
    """d x as two bf16 numbers holds 16 bits: the error in norm is that of rounding the 64-bit gradient, and 2^-16 / 2^-9 of it."""
    from hawk_b200 import linear_logprobs
    for seed in range(4):
        w, a, t, gl, ge = _case(N, 96, 5802, seed)
        _, _, dw, _ = _reference(w, a, t, gl, ge)
        w.requires_grad_()
        out = linear_logprobs(w, torch.cat((a, a)), torch.cat((t, torch.full_like(t, -1))))  # as many rows again left out
        got, = torch.autograd.grad(out, w, (torch.cat((gl, gl)), torch.cat((ge, ge))))
        assert rel_l2(got, dw) <= 1.05 * rel_l2(dw.bfloat16(), dw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wanted", [(True, True), (True, False), (False, True)])
def test_a_failure_shows_in_the_results(wanted, dtype):
    """The status word as a kernel leaves it that gave up a wait (set here by hand): results and gradients are NaN, the check
    raises once, and what follows is right again."""
    from hawk_b200 import check_device_status, ops
    w, a, t, gl, ge = _case(70, 64, 300, 17, dtype)
    t[::3] = -1
    lp, H, saved = ops.linear_logprobs_fwd(w, a, t, True)
    good = ops.linear_logprobs_bwd(w, a, t, saved, lp, H, gl, ge, *wanted)
    ops._status_word(w.device).fill_(1)
    try:
        bad = ops.linear_logprobs_fwd(w, a, t, True)
        assert bool(bad[0][t >= 0].isnan().all()) and bool(bad[1][t >= 0].isnan().all())
        dw, da = ops.linear_logprobs_bwd(w, a, t, saved, lp, H, gl, ge, *wanted)
        assert not wanted[0] or bool(dw[0, 0].isnan())
        assert not wanted[1] or (bool(da[t >= 0].isnan().all()) and bool((da[t < 0] == 0).all()))
        with pytest.raises(RuntimeError, match="abandoned"):
            check_device_status()
    finally:
        ops._status_word(w.device).zero_()
    check_device_status()
    again = ops.linear_logprobs_bwd(w, a, t, saved, lp, H, gl, ge, *wanted)
    assert all(torch.equal(x, y) for x, y in zip(good, again))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [8192, 8193])
def test_activations_gradient_of_many_rows(N, dtype):
    """Both sides of where its splits are planned on the device, few and many of the rows named, fp32 and bf16 results."""
    w, a, t, gl, ge = _case(N, 64, 1000, 18, dtype)
    for every in (1, 2, 40):
        _check(w, a, torch.where(torch.arange(N, device="cuda") % every == 0, t, -1), gl, ge)


@pytest.mark.parametrize("w_dtype", [F32, BF16])
@pytest.mark.parametrize("N", [100, 129, 255, 1548])
def test_gradients_of_a_mean(N, w_dtype):
    """Upstream gradients alike in every row: no rounding may turn into a common factor.  With N >= 100 rows, H = 64 and 2000 tokens the
    weight's gradient takes at least N H = 6400 independent roundings of at most 2^-8, so its component along the true one is off by
    2^-8 / sqrt(3 N H) = 3e-5 in the mean square; 2^-11 is 17 times that.  As a whole it is off by two roundings of operands and, in bf16,
    its own: sqrt(3) 2^-8 / sqrt(3) in norm at most."""
    from hawk_b200 import linear_logprobs
    w, a, t, _, _ = _case(N, 64, 2000, N, w_dtype=w_dtype, lift=0.0)
    w, a = w.detach().requires_grad_(), a.detach().requires_grad_()
    lp, H = linear_logprobs(w, a, t)
    gl = torch.full((N,), -1.0 / N, device="cuda")
    dw, da = torch.autograd.grad(lp, (w, a), gl)
    _, _, rdw, rda = _reference(w.detach(), a.detach(), t, gl, torch.zeros_like(gl))
    named = torch.zeros(2000, dtype=torch.bool, device="cuda").index_fill_(0, t, True)
    for got, want in ((dw[named], rdw[named]), (dw[~named], rdw[~named]), (da, rda)):
        factor = float((got.double() * want).sum() / (want * want).sum())
        assert abs(factor - 1) <= 2.0 ** -11, factor
        assert rel_l2(got, want) <= 2.0 ** -8


@pytest.mark.parametrize("want", [True, False])
@pytest.mark.parametrize("lift,V", [(30.0, 1000), (30.0, 129), (45.0, 32000)])
def test_all_but_certain_tokens(lift, V, want):
    """1 - p and the entropy of tokens whose probability rounds to 1, against their own size.  Each logit is off by 2^-20 of the logits' spread
    and by half a step of fp32, and a term by twice that; 64 terms added one after the other, their two sums, and 13 such sums of groups are
    77 roundings of 2^-24 (with log1p's 2^-17).  They are relative to 1 - p where it is below 2^-9: its even and odd columns' maxima are
    further apart than that, and the token's 1 is not in the sum; else to a sum of up to 2, which leaves 77 2^-24 / (1 - p)."""
    from hawk_b200 import linear_logprobs
    w, a, t, gl, ge = _case(384, 256, V, V, lift=lift)
    w.requires_grad_(want)
    lp, H = (x.detach().double() for x in linear_logprobs(w, a, t))
    logits = a.double() @ w.detach().double().T
    x = logits.gather(1, t[:, None])
    others = (logits - x).scatter(1, t[:, None], -math.inf)
    tail = others.exp().sum(1)                      # (1 - p) / p
    q = torch.log1p(tail)                           # -log p
    entropy = q + (torch.where(others.isinf(), 0.0, others) * -(others - q[:, None]).exp()).sum(1)
    sure = (tail < 0.1) & (tail > 1e-25)
    assert int(sure.sum()) > 100 and int((tail[sure] < 1e-7).sum()) > 30
    bound = 2 * (float(logits.abs().max()) * (2.0 ** -20 + 2.0 ** -24)) + 2.0 ** -17 + torch.where(tail < 2.0 ** -9, 0.0, 77 * 2.0 ** -24 / tail)
    assert bool(((torch.expm1(-lp) / tail - 1).abs() <= bound)[sure].all())
    assert bool(((H / entropy - 1).abs() <= 2 * bound)[sure].all())  # its terms hold the logarithm as well
