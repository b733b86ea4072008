"""The global gradient norm, clipping and the clipped optimiser step against the same in 64 bits.

Tolerances: the norm is one fp32 rounding of a sum whose terms are right to 8 roundings of 2^-24 each, summed in double:
under 1e-6 relative.  A clipped gradient is the rounding of g * coef, coef itself rounded: 2 * eps / 2 of the type plus
2^-24; an AdamW step on fp32 tensors is held to the bound of its own test."""
import math

import pytest
import torch

from conftest import rel_l2

pytestmark = pytest.mark.gpu


def _list(seed, dtypes=(torch.float32, torch.bfloat16), count=40):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i in range(count):
        n = [1, 7, 8, 255, 8191, 8192, 8193, 16385, 100003, 513 * 129][i % 10]
        out.append((torch.randn(n, generator=g, device="cuda") * 10.0 ** (i % 5 - 3)).to(dtypes[i % len(dtypes)]))
    return out


def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


@pytest.mark.parametrize("count", [1, 2, 40, 128, 129, 1023, 1024, 1025, 2100])
def test_norm_of_lists(count):
    from hawk_b200 import grad_norm
    ts = _list(count, count=count)
    got = grad_norm(ts)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(float(got) - _norm64(ts)) <= 1e-6 * _norm64(ts)
    assert torch.equal(got, grad_norm(ts))


def test_norm_of_views_and_empty_tensors():
    from hawk_b200 import grad_norm
    base = torch.randn(3000, 7, device="cuda")
    ts = [base[1:].view(-1)[1:], base.t(), base[::3], torch.empty(0, device="cuda"), base.bfloat16().view(-1)[3:]]
    assert abs(float(grad_norm(ts)) - _norm64(ts)) <= 1e-6 * _norm64(ts)
    assert float(grad_norm([torch.empty(0, 4, device="cuda")])) == 0.0
    assert float(grad_norm([torch.zeros(9, device="cuda")])) == 0.0
    assert abs(float(grad_norm(base)) - _norm64([base])) <= 1e-6 * _norm64([base])  # a tensor by itself


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e18, 1e30, 1e37])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_beyond_the_range_of_squares(scale, dtype):
    from hawk_b200 import grad_norm
    t = (torch.rand(5001, device="cuda") * scale).to(dtype)
    got, norm = float(grad_norm([t])), _norm64([t])
    # 5001 values of 1e37 have a norm of sqrt(5001 / 3) 1e37 = 4.1e38, above fp32's largest 3.403e38: its rounding is infinity
    want = float(torch.tensor(norm, dtype=torch.float64).float())
    assert got == want if math.isinf(want) else abs(got - norm) <= 1e-6 * norm


def test_norm_of_non_finite_values():
    from hawk_b200 import grad_norm
    a, b = torch.randn(100, device="cuda"), torch.randn(33000, device="cuda").bfloat16()
    b[32999] = math.inf
    assert float(grad_norm([a, b])) == math.inf
    a[3] = math.nan
    assert math.isnan(float(grad_norm([a, b])))


@pytest.mark.parametrize("share", [0.0, 0.25, 2.0, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clip_matches_the_rule(share, dtype):
    from hawk_b200.train import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(t.shape, dtype=dtype, device="cuda")) for t in _list(3)]
    for p, t in zip(ps, _list(3)):
        p.grad = t.to(dtype)
    ps.append(torch.nn.Parameter(torch.zeros(70, 30, dtype=dtype, device="cuda")))
    ps[-1].grad = torch.randn(30, 70, device="cuda").to(dtype).t()   # a gradient that is not contiguous
    ps.append(torch.nn.Parameter(torch.zeros(3, device="cuda")))     # and a parameter without one
    had = [p.grad.clone() for p in ps[:-1]]
    norm = _norm64(had)
    version = ps[0].grad._version
    got = clip_grad_norm_(ps + ps[:1], share * norm)                 # a parameter named twice counts once
    assert abs(float(got) - norm) <= 1e-6 * norm and ps[0].grad._version > version
    coef = min(1.0, share * norm / (norm + 1e-6))
    for p, h in zip(ps, had):
        if coef == 1.0:
            assert torch.equal(p.grad, h)
        else:
            bound = torch.finfo(dtype).eps / 2 + 4 * 2.0 ** -24
            assert bool(((p.grad.double() - h.double() * coef).abs() <= bound * (h.double() * coef).abs() + 1e-38).all())


def test_clip_makes_every_gradient_nan_when_one_is():
    from hawk_b200.train import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(5, device="cuda")) for _ in range(2)]
    ps[0].grad, ps[1].grad = torch.ones(5, device="cuda"), torch.full((5,), math.nan, device="cuda")
    assert math.isnan(float(clip_grad_norm_(ps, 1.0))) and bool(ps[0].grad.isnan().all())  # as torch's


def test_refusals():
    from hawk_b200 import grad_norm, ops
    from hawk_b200.train import FusedAdamW, clip_grad_norm_
    a = torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="CUDA"):
        grad_norm([a, torch.ones(3)])
    with pytest.raises(TypeError, match="float16"):
        grad_norm([a.half()])
    with pytest.raises(ValueError, match="share memory"):
        ops.scale_in_place([a, a[2:]], torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="scalar"):
        ops.scale_in_place([a], torch.ones(2, device="cuda"))
    p = torch.nn.Parameter(a)
    p.grad = a.clone()
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
        with pytest.raises(ValueError, match="max_grad_norm"):
            FusedAdamW([p], max_grad_norm=bad)


@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_clipped_adamw_matches_torch(max_norm):
    from hawk_b200.train import FusedAdamW
    shapes = [(33, 65), (8193,), (4, 128), (1,)]
    torch.manual_seed(0)
    ours = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    ref = [torch.nn.Parameter(p.detach().double().clone()) for p in ours]
    groups = lambda ps: [dict(params=ps[:2]), dict(params=ps[2:], lr=1e-2)]  # noqa: E731
    opt = FusedAdamW(groups(ours), lr=1e-3, weight_decay=0.1, max_grad_norm=max_norm)
    topt = torch.optim.AdamW(groups(ref), lr=1e-3, weight_decay=0.1)
    for _ in range(4):
        for p, q in zip(ours, ref):
            g = torch.randn(p.shape, device="cuda")
            p.grad, q.grad = g, g.double()
        norm = torch.nn.utils.clip_grad_norm_(ref, max_norm)
        kept = [p.grad.clone() for p in ours]
        opt.step()
        topt.step()
        assert abs(float(opt.grad_norm) - float(norm)) <= 1e-6 * float(norm)
        assert all(torch.equal(p.grad, k) for p, k in zip(ours, kept))  # the gradients stay as they were
    for p, q in zip(ours, ref):
        assert rel_l2(p.detach(), q.detach()) <= 2e-6


def test_unclipped_adamw_is_unchanged_by_a_large_bound():
    from hawk_b200.train import FusedAdamW
    torch.manual_seed(1)
    a = [torch.nn.Parameter(torch.randn(5000, device="cuda")) for _ in range(3)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    oa, ob = FusedAdamW(a), FusedAdamW(b, max_grad_norm=1e30)
    for p, q in zip(a, b):
        p.grad = q.grad = torch.randn(5000, device="cuda")
    oa.step()
    ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and oa.grad_norm is None


def test_captured_norm_follows_its_inputs():
    from hawk_b200 import grad_norm
    ts = _list(9, count=130)
    grad_norm(ts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grad_norm(ts)
    for k in (1.0, 3.0):
        for t in ts:
            t.mul_(k)
        graph.replay()
        assert abs(float(got) - _norm64(ts)) <= 1e-6 * _norm64(ts)


def test_norm_on_another_stream():
    from hawk_b200 import grad_norm
    ts = _list(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in ts:
            t.mul_(2.0)
        got = grad_norm(ts)
    torch.cuda.current_stream().wait_stream(side)
    assert abs(float(got) - _norm64(ts)) <= 1e-6 * _norm64(ts)


def test_trainer_clips():
    import hawk_b200.model as M
    from hawk_b200.train import Trainer
    cfg = M.HawkConfig(96, 64, 128, 2, 64, 4, 4)
    ids = torch.randint(1, 96, (2, 33), device="cuda")
    tr = Trainer(cfg, "cuda", seed=3, max_grad_norm=0.25)
    grads = []
    tr.step(ids, after_backward=lambda _: grads.extend(p.grad.clone() for p in tr.model.parameters()))
    assert abs(float(tr.grad_norm) - _norm64(grads)) <= 1e-6 * _norm64(grads)
    first = next(p for p in tr.model.parameters() if p.dim() == 2)
    st = tr.opt.state[first]
    coef = min(1.0, 0.25 / (_norm64(grads) + 1e-6))
    assert rel_l2(st["exp_avg"], 0.1 * coef * grads[0].double()) <= 1e-6


def test_a_step_without_gradients_has_no_norm():
    from hawk_b200 import train
    p = torch.nn.Parameter(torch.ones(100, device="cuda"))
    opt = train.FusedAdamW([p], max_grad_norm=1.0)
    p.grad = torch.ones_like(p)
    opt.step()
    assert float(opt.grad_norm) == 10.0
    p.grad = None
    opt.step()
    assert opt.grad_norm is None


def test_a_refused_clip_changes_nothing():
    from hawk_b200 import train
    ps = [torch.nn.Parameter(torch.zeros(n, n, device="cuda")) for n in (8, 8, 6)]
    ps[0].grad = ps[1].grad = torch.ones(8, 8, device="cuda")  # one tensor as the gradient of two parameters
    ps[2].grad = torch.ones(6, 12, device="cuda")[:, ::2]
    with pytest.raises(ValueError, match="share memory"):
        train.clip_grad_norm_(ps, 0.5)
    assert all(bool((p.grad == 1).all()) for p in ps)


def test_norm_of_nothing_can_be_captured():
    from hawk_b200 import grad_norm
    empty = [torch.empty(0, device="cuda"), torch.empty(3, 0, device="cuda")]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = grad_norm(empty)
    graph.replay()
    assert norm.is_cuda and float(norm) == 0.0 and float(grad_norm([])) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 7, 8, 9, 8192, 16384, 16391, 100003])
def test_views_of_a_flat_buffer(n, dtype):
    """Every distance from a 16-byte boundary; what lies before and behind a view is neither counted nor written."""
    from hawk_b200 import grad_norm, ops
    g = torch.Generator(device="cuda").manual_seed(n)
    for off in range(8):
        flat = torch.full((n + 24,), float("nan"), device="cuda", dtype=dtype)
        v = flat[off:off + n]
        v.copy_(torch.randn(n, generator=g, device="cuda"))
        want = v.double()
        assert abs(float(grad_norm([v])) - float(want.norm())) <= 1e-6 * float(want.norm())
        ops.scale_in_place([v], torch.tensor(0.37, device="cuda"))
        half = torch.finfo(dtype).eps / 2
        assert bool(((v.double() - want * 0.37).abs() <= (half + 2 * 2.0 ** -24) * want.abs() * 0.37).all())
        assert bool(flat[:off].isnan().all()) and bool(flat[off + n:].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_gradients_get_the_same_factor(dtype):
    """A factor that bf16 does not hold (0.37), on gradients of every layout: one rounding each."""
    from hawk_b200.train import clip_grad_norm_
    torch.manual_seed(2)
    flat = torch.randn(40, 96, device="cuda").to(dtype)
    ps = [torch.nn.Parameter(torch.zeros(s, dtype=dtype, device="cuda")) for s in ((40, 32), (40, 32), (48, 33), (7, 5, 3), (0, 4))]
    ps[0].grad, ps[1].grad = flat[:, ::3], flat[:, 1::3]  # interleaved, but without an element in common
    ps[2].grad = torch.randn(33, 48, device="cuda").to(dtype).t()
    ps[3].grad = torch.randn(3, 5, 7, device="cuda").to(dtype).permute(2, 1, 0)
    ps[4].grad = torch.zeros(4, 0, dtype=dtype, device="cuda").t()
    had, between = [p.grad.clone() for p in ps], flat[:, 2::3].clone()
    norm = _norm64(had)
    layouts = [(p.grad.data_ptr(), p.grad.stride(), p.grad._version) for p in ps[:4]]
    assert abs(float(clip_grad_norm_(ps, 0.37 * norm)) - norm) <= 1e-6 * norm
    for p, h, (at, stride, version) in zip(ps, had, layouts):
        want = h.double() * (0.37 * norm / (norm + 1e-6))
        assert bool(((p.grad.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 4 * 2.0 ** -24) * want.abs()).all())
        assert (p.grad.data_ptr(), p.grad.stride()) == (at, stride) and p.grad._version > version
    assert torch.equal(flat[:, 2::3], between)


def test_strided_gradients_that_share_memory_are_scaled_once():
    from hawk_b200.train import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(8, 8, device="cuda")) for _ in range(3)]
    shared = torch.ones(8, 8, device="cuda").t()
    flat = torch.ones(8, 8, device="cuda")
    shared[0, 1] = 2.0  # not its own transpose
    ps[0].grad = ps[1].grad = shared
    ps[2].grad = torch.ones(8, 16, device="cuda")[:, ::2]
    more = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in ((8, 8), (4, 8))]
    more[0].grad, more[1].grad = flat, flat[::2]  # a contiguous one and a strided view of it
    had = [p.grad.clone() for p in ps + more]
    norm = _norm64(had)
    clip_grad_norm_(ps + more, norm / 4)
    for p, h in zip(ps + more, had):
        assert torch.allclose(p.grad, h * 0.25, rtol=1e-6)


def test_a_clip_that_cannot_be_written_changes_nothing():
    from hawk_b200.train import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(8, 8, device="cuda")) for _ in range(2)]
    ps[0].grad, ps[1].grad = torch.ones(8, 8, device="cuda"), torch.ones(8, 1, device="cuda").expand(8, 8)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(ps, 0.5)
    assert all(bool((p.grad == 1).all()) for p in ps)


def test_a_factor_among_the_scaled_is_refused():
    from hawk_b200 import ops
    x = torch.full((9,), 2.0, device="cuda")
    for ts, scale in (([x], x[3]), ([x], x[:1]), ([torch.ones(4, device="cuda"), x], x[8])):
        with pytest.raises(ValueError, match="share memory"):
            ops.scale_in_place(ts, scale)
    ops.scale_in_place([x[:8]], x[8])  # beside it is well
    assert x.tolist() == [4.0] * 8 + [2.0]


def test_every_adamw_entry_point_forms_the_same_update():
    import struct

    from hawk_b200 import _lib
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    torch.manual_seed(4)
    first = [torch.randn(1000, device="cuda") for _ in range(2)] + [torch.zeros(1000, device="cuda") for _ in range(2)]
    rest = (1e-3, 0.9, 0.999, 1e-8, 0.1)
    got = []
    for entry in ("scaled", "multi", "step"):
        p, g, m, v = (t.clone() for t in first)
        for step in (1, 2, 3):
            one = struct.pack("6Q", *(t.data_ptr() for t in (p, g, m, v)), 0, 1000)
            if entry == "scaled":
                rc = lib.hawk_adamw_multi_scaled(one, 1, *rest, step, None, st)
            elif entry == "multi":
                rc = lib.hawk_adamw_multi(one, 1, *rest, step, st)
            else:
                rc = lib.hawk_adamw_step(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), None, 1000, *rest, step, st)
            assert rc == 0
        got.append((p, m, v))
    g = first[1].double()
    # v after three equal gradients: g^2 (1 - beta^3), three roundings a step
    assert float((got[0][2].double() / (g * g * (1 - 0.999 ** 3)) - 1).abs().max()) <= 12 * 2.0 ** -24
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
