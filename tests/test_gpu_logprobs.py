"""Log probabilities, entropy, alternatives and the logits' gradient against plain ones in 64 bits.

Tolerances.  d = x - m is rounded once (2^-24 |d|), exp2 of d log2 e is off by 2^-22 + 2^-23 |d| log2 e relative; only terms with
|d| < 20 or so count in the sums, which are tree sums of depth < 64: log s is off by less than 30 * 2^-22 = 8e-6 absolute, a log
probability by 2^-23 of its size more, the entropy (sum of p |d|) by 3e-5 relative to 1 + H.  The gradient: p is off by
2^-22 + (|log p| + 8) 2^-22 relative, the factor (log p + H) by 1e-5 absolute; then one rounding to the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _reference(logits, tokens, top):
    x = logits.double()
    V = x.shape[-1]
    named = tokens >= 0
    lse = torch.logsumexp(x, -1)
    logp = x - lse[..., None]
    p = logp.exp()
    H = -(torch.where(p > 0, p * logp, 0)).sum(-1)
    at = tokens.clamp(0, V - 1)[..., None]
    lp = torch.where(tokens < V, logp.gather(-1, at)[..., 0], math.nan)
    ids = x.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    return (torch.where(named, lp, 0), torch.where(named, H, 0), torch.where(named[..., None], logp.gather(-1, ids), -math.inf),
            torch.where(named[..., None], ids, -1), logp, p, H, named)


def _check(logits, tokens, top):
    from hawk_b200 import token_logprobs
    lp, H, best, ids = token_logprobs(logits, tokens, top)
    rlp, rH, rbest, rids, *_ = _reference(logits.detach(), tokens, top)
    assert lp.dtype == H.dtype == best.dtype == F32 and ids.dtype == torch.int64
    assert lp.shape == H.shape == tokens.shape and best.shape == ids.shape == (*tokens.shape, top)
    assert torch.equal(ids, rids)
    close = lambda a, b, tol: bool(((a.double() - b).abs() <= tol).logical_or(a.double() == b).all())  # noqa: E731
    assert close(lp, rlp, 8e-6 + 2.0 ** -22 * rlp.abs())
    assert close(H, rH, 3e-5 * (1 + rH))
    assert close(best, rbest, 8e-6 + 2.0 ** -22 * rbest.abs())
    return lp, H, best, ids


def _check_gradient(dx, x, t, gl, ge):
    *_, logp, p, rH, named = _reference(x, t, 0)
    gl, ge = gl.double(), ge.double()
    hot = torch.zeros_like(logp).scatter_(-1, t.clamp(min=0)[..., None], 1.0)
    factor = gl[..., None] + ge[..., None] * (logp + rH[..., None])
    want = torch.where(named[..., None], gl[..., None] * hot - p * factor, 0)
    off = p * (factor.abs() * (logp.abs() + 10) * 2.0 ** -21 + ge.abs()[..., None] * 4e-5 * (1 + rH[..., None]))
    off = off + hot * gl.abs()[..., None] * (1e-5 * (1 - p).clamp(min=1e-9) + 2.0 ** -22 * (1 - p) + 1.6e-5 * p)
    assert bool(((dx.double() - want).abs() <= off + torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 1e-3) + 1e-37).all())


def _case(rows, V, dtype, seed=0, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (scale * torch.randn(rows, V, generator=g, device="cuda")).to(dtype)
    return x, torch.randint(0, V, (rows,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V", [(1, 1), (1, 2), (3, 7), (2, 8), (5, 63), (1, 4095), (7, 4096), (2, 4097), (300, 513), (1, 32000),
                                    (256, 32000), (3, 31999), (77, 16385), (149, 32768), (2, 65537), (400, 65536), (1, 131072),
                                    (2, 262147), (1, 300001), (160, 40001)])
def test_values_and_alternatives(rows, V, dtype):
    x, t = _case(rows, V, dtype, rows + V)
    for top in sorted({0, min(1, V), min(5, V), min(20, V), min(32, V)}):
        _check(x, t, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [33, 8191, 32000, 140000])
def test_ties_and_order(V, dtype):
    """Rows whose candidates are many: all equal, rising, falling, two values, few distinct ones."""
    n = torch.arange(V, device="cuda")
    rows = [torch.zeros(V, device="cuda"), n / 64, -n / 64, (n % 7 == 3).float(), (n % 3).float() - 1, (n == V - 1).float() * 9,
            torch.where(n < 40, 1.0, 1.0 + (n % 2) / 128), (n // 5 % 100).float(),
            torch.where(n % 2 == 0, -0.0, 0.0), torch.where(n % 3 == 0, -0.0, torch.where(n % 3 == 1, 0.0, -1.0))]
    x = torch.stack(rows).to(dtype)
    for top in (1, 17, 32):
        _check(x, torch.full((len(rows),), V // 2, device="cuda"), top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [50, 32000, 100003])
def test_masked_rows(V, dtype):
    from hawk_b200 import token_logprobs
    lowest = torch.finfo(dtype).min
    x, t = _case(6, V, dtype, V)
    for fill in (-math.inf, lowest):
        y = torch.full_like(x, fill)
        keep = torch.tensor([0, 3, V // 2, V - 1], device="cuda")
        y[:5, keep] = x[:5, keep]
        t[:4] = keep
        t[4] = 1            # a token that cannot come
        y[5, 7] = x[5, 7]   # one that has to
        t[5] = 7
        lp, H, best, ids = token_logprobs(y, t, 20)
        r = _reference(y, t, 20)
        assert torch.equal(ids, r[3])
        assert float(lp[5]) == 0 and float(H[5]) == 0
        if fill == -math.inf:
            assert float(lp[4]) == -math.inf and bool((best[:5, 4:] == -math.inf).all())
        else:
            assert float(lp[4]) < -1e38
        assert torch.allclose(lp[:4].double(), r[0][:4], atol=1e-5, rtol=1e-6) and torch.allclose(H.double(), r[1], atol=1e-5, rtol=1e-5)
    y = torch.full_like(x, lowest)  # all alike: a uniform row
    lp, H, best, ids = token_logprobs(y, t, 4)
    assert torch.allclose(lp, torch.full_like(lp, -math.log(V)), rtol=1e-5) and torch.allclose(H, torch.full_like(H, math.log(V)), rtol=1e-5)
    assert ids.tolist() == [[0, 1, 2, 3]] * 6


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [40, 32000, 70001])
def test_rows_left_out_empty_and_spoilt(V, dtype):
    from hawk_b200 import token_logprobs
    x, t = _case(8, V, dtype, 3)
    x[0] = math.nan                   # left out, whatever it holds
    x[1] = math.inf
    t[0], t[1] = -1, -2 ** 40
    x[2] = -math.inf                  # nothing can come
    x[3, 5] = math.nan
    x[4] = math.nan
    x[5, V - 1] = math.inf
    t[6] = V
    x = x.requires_grad_()
    lp, H, best, ids = token_logprobs(x, t, 3)
    assert lp[:2].tolist() == H[:2].tolist() == [0, 0] and bool((best[:2] == -math.inf).all()) and bool((ids[:2] == -1).all())
    assert float(lp[2]) == -math.inf and float(H[2]) == 0 and ids[2].tolist() == [0, 1, 2] and bool((best[2] == -math.inf).all())
    assert bool(lp[3:6].isnan().all()) and bool(H[3:6].isnan().all())
    others = x.detach()[3].double()
    others[5] = -math.inf
    assert torch.equal(ids[3], others.sort(descending=True, stable=True).indices[:3])
    assert ids[4].tolist() == [-1] * 3 and int(ids[5, 0]) == V - 1
    assert math.isnan(float(lp[6])) and math.isfinite(float(H[6])) and math.isfinite(float(lp[7]))
    dx, = torch.autograd.grad(lp[[0, 1, 2, 6, 7]].sum() + H[[0, 1, 2, 7]].sum(), x)
    assert float(dx[:3].abs().max()) == 0 and bool(dx[6].isnan().all()) and bool(dx[7].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [1e4, -3e4, 6e4])
def test_far_offsets(shift, dtype):
    """Softmax does not see a common offset; x - m is exact for values this near one another."""
    x, t = _case(4, 1000, F32, 1)
    x = (x * 64).round() / 64 + shift
    _check(x.to(dtype), t, 8)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 7), (2, 1024), (5, 1025), (9, 32000), (4, 31999), (2, 100003)])
@pytest.mark.parametrize("which", ["both", "logprob", "entropy"])
def test_gradient(rows, V, dtype, which):
    from hawk_b200 import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(rows + V)
    x, t = _case(rows, V, dtype, rows * V)
    x[0, t[0]] += 25  # a token that is all but certain
    if rows > 2:
        t[1] = -1
    x = x.requires_grad_()
    lp, H, *_ = token_logprobs(x, t)
    gl, ge = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    use = dict(both=((lp, H), (gl, ge)), logprob=((lp,), (gl,)), entropy=((H,), (ge,)))[which]
    dx, = torch.autograd.grad(use[0], x, use[1])
    _check_gradient(dx, x.detach(), t, gl * (which != "entropy"), ge * (which != "logprob"))


def test_gradient_against_differences():
    """Central differences of the 64-bit function at a few logits; the kernel's gradient in fp32."""
    from hawk_b200 import token_logprobs
    x, t = _case(3, 50, F32, 4)
    x = x.requires_grad_()
    lp, H, *_ = token_logprobs(x, t)
    dx, = torch.autograd.grad((lp * 1.5 - 0.5 * H).sum(), x)
    f = lambda z: (1.5 * _reference(z, t, 0)[0] - 0.5 * _reference(z, t, 0)[1]).sum()  # noqa: E731
    for r, j in [(0, 0), (1, int(t[1])), (2, 49)]:
        e = torch.zeros(3, 50, dtype=torch.float64, device="cuda")
        e[r, j] = 1e-4
        assert abs(float((f(x.detach().double() + e) - f(x.detach().double() - e)) / 2e-4) - float(dx[r, j])) <= 1e-5


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_of_logits(dtype):
    from hawk_b200 import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(7)
    base = torch.randn(4, 6, 1001, generator=g, device="cuda").to(dtype)
    views = [base[:, -1], base[:, 2:4], base[..., 1:], base[:, 1, 3:900], base[:, :, ::2], base.transpose(0, 1), base[0, 0], base[:1, :1],
             base[:, :1].expand(4, 3, 1001)]
    for v in views:
        t = torch.randint(0, v.shape[-1], v.shape[:-1], generator=g, device="cuda")
        leaf = v.detach()
        _check(leaf, t, 6)
        leaf = leaf.requires_grad_()
        # not the bits of a contiguous copy's: where a row starts decides which thread adds which of its elements
        ones = torch.ones(t.shape, device="cuda")
        _check_gradient(torch.autograd.grad(sum(o.sum() for o in token_logprobs(leaf, t, 2)[:2]), leaf)[0], v, t, ones, ones)
    lp, H, best, ids = token_logprobs(base[:, :0], torch.zeros(4, 0, dtype=torch.int64, device="cuda"), 2)
    assert lp.shape == (4, 0) and ids.shape == (4, 0, 2)
    assert not best.requires_grad and token_logprobs(base, torch.zeros(4, 6, dtype=torch.int32, device="cuda"))[0].shape == (4, 6)


def test_alternatives_carry_no_gradient():
    from hawk_b200 import token_logprobs
    x, t = _case(2, 64, F32)
    lp, H, best, ids = token_logprobs(x.requires_grad_(), t, 4)
    assert lp.requires_grad and H.requires_grad and not best.requires_grad


def test_neighbouring_rows_are_untouched():
    """Rows behind the last and elements beside a view's rows keep what they held."""
    from hawk_b200 import ops
    import hawk_b200._lib as L
    lib = L.load()
    x, t = _case(3, 1003, BF16)
    out = torch.full((5, 1003), 77.0, dtype=BF16, device="cuda")
    lp, H, _, _, stats = ops.token_logprobs_fwd(x, t, 0)
    assert lib.hawk_token_logprobs_bwd(x.data_ptr(), 1003, t.data_ptr(), stats.data_ptr(), lp.data_ptr(), H.data_ptr(), lp.data_ptr(),
                                       None, out[1].data_ptr(), 3, 1003, 1, torch.cuda.current_stream().cuda_stream) == 0
    assert bool((out[0] == 77).all()) and bool((out[4] == 77).all()) and bool((out[1:4] != 77).all())


def test_refusals():
    from hawk_b200 import token_logprobs
    x, t = _case(3, 10, F32)
    for top in (-1, 11, 33):
        with pytest.raises(ValueError, match="top"):
            token_logprobs(x, t, top)
    with pytest.raises(ValueError, match="shape"):
        token_logprobs(x, t[:2])
    with pytest.raises(TypeError, match="integers"):
        token_logprobs(x, t.float())
    with pytest.raises(TypeError, match="float16"):
        token_logprobs(x.half(), t)
    with pytest.raises(RuntimeError, match="cpu"):
        token_logprobs(x, t.cpu())


def test_captured():
    from hawk_b200 import token_logprobs
    x, t = _case(5, 32000, BF16, 8)
    token_logprobs(x, t, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, t, 5)
    y, u = _case(5, 32000, BF16, 9)
    x.copy_(y)
    t.copy_(u)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, token_logprobs(y, u, 5)))
