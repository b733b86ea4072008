"""The embedding and its gradient by token against plain ones in 64 bits.

Tolerances.  Forward: one product rounded to fp32 and, in bf16, once more: eps / 2 of the type plus 2^-24, relative.
Gradient: a sum of c rows in fp32 in order, at most (c - 1) 2^-24 sum |row| off, times the scale (2^-24), rounded to the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _zipf(n, V, g):
    return (float(V) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).long().sub_(1).clamp_(0, V - 1)


def _check(ids, V, H, dtype, scale=1.0, padding=None, seed=0):
    from hawk_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, H, generator=g, device="cuda").to(dtype).requires_grad_()
    out = embedding(ids, w, scale, padding)
    assert out.shape == (*ids.shape, H) and out.dtype == dtype
    half = torch.finfo(dtype).eps / 2
    want = w.detach().double()[ids] * scale
    assert bool(((out.double() - want).abs() <= (half + 2.0 ** -24) * want.abs()).all())
    go = torch.randn(out.shape, generator=g, device="cuda").to(dtype)
    dw, = torch.autograd.grad(out, w, go, retain_graph=True)
    again, = torch.autograd.grad(out, w, go)
    assert dw.dtype == dtype and torch.equal(dw, again)
    flat, rows = ids.reshape(-1), go.reshape(-1, H).double()
    if padding is not None:
        rows = torch.where((flat == padding % V)[:, None], 0, rows)
    sums = torch.zeros(V, H, dtype=torch.float64, device="cuda").index_add_(0, flat, rows)
    mags = torch.zeros(V, H, dtype=torch.float64, device="cuda").index_add_(0, flat, rows.abs())
    counts = torch.zeros(V, dtype=torch.float64, device="cuda").index_add_(0, flat, torch.ones_like(flat, dtype=torch.float64))
    bound = (half + 2.0 ** -23) * (sums * scale).abs() + counts[:, None] * 2.0 ** -24 * mags * abs(scale) * (1 + 2 * half)
    assert bool(((dw.double() - sums * scale).abs() <= bound).all())
    assert bool((dw[counts == 0] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,H", [(1, 1, 1), (1, 300, 64), (31, 7, 5), (64, 1, 24), (65, 1, 24), (129, 3, 2), (1551, 32000, 512),
                                   (4097, 1000, 2048), (8192, 50, 36), (8193, 129, 250), (20000, 5000, 1001), (3000, 70001, 8)])
def test_embedding_matches(n, V, H, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + V + H)
    _check(_zipf(n, V, g), V, H, dtype, scale=1.0 if n % 2 else 22.6)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [16, 31, 32, 33, 47, 48, 49, 63, 64, 65, 96, 97, 8191, 8192, 8193, 40000])
def test_one_token_everywhere(n, dtype):
    """All positions of one block's slice, past its queue; runs that end inside, at and after a window."""
    _check(torch.full((n,), 11, device="cuda"), 40, 72, dtype)


@pytest.mark.parametrize("lead", [0, 1, 15, 16, 17, 31, 32, 33, 63])
def test_runs_across_windows(lead):
    ids = torch.cat([torch.zeros(lead, dtype=torch.int64), torch.full((200,), 5), torch.full((64,), 6), torch.full((65,), 8),
                     torch.arange(9, 30)]).cuda()
    _check(ids, 30, 40, F32)
    _check(ids[torch.randperm(ids.numel(), device="cuda")].view(1, -1), 30, 40, BF16)


def test_every_vocabulary_slice_width():
    for V in (31, 32, 33, 147 * 32, 148 * 32 + 1, 148 * 100 + 3, 148 * 4096 + 17):
        g = torch.Generator(device="cuda").manual_seed(V)
        _check(torch.randint(0, V, (777,), generator=g, device="cuda"), V, 4, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padding_and_strangers(dtype):
    from hawk_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = _zipf(999, 200, g).view(3, 333)
    _check(ids, 200, 33, dtype, scale=0.5, padding=0)
    _check(ids, 200, 32, dtype, padding=-200)
    w = torch.randn(10, 16, device="cuda").to(dtype).requires_grad_()
    odd = torch.tensor([3, -1, 10, 2 ** 40, 9, -2 ** 62], device="cuda")
    out = embedding(odd, w)
    assert out.isnan().all(1).tolist() == [False, True, True, True, False, True]
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert dw.sum(1).tolist() == [16.0 if i in (3, 9) else 0.0 for i in range(10)]


def test_strides_types_and_empty_calls():
    from hawk_b200 import embedding
    base = torch.randn(51, 40, device="cuda")
    ids = torch.randint(0, 50, (6, 10), device="cuda")
    for w in (base[:50], base[1:], base[:50, :39], base.view(-1)[1:2001].view(50, 40), base.t()[:, :40]):  # odd addresses and strides
        w = w.detach().requires_grad_()
        k = ids % w.shape[0]
        out = embedding(k.t(), w, 2.0)
        assert torch.equal(out, w.detach()[k.t()] * 2.0)
        dw, = torch.autograd.grad(out, w, torch.ones(1, device="cuda").expand(out.shape))  # a broadcast gradient
        assert torch.equal(dw[:, 0], 2.0 * torch.bincount(k.view(-1), minlength=w.shape[0]).float())
    w = base.detach().requires_grad_()
    assert torch.equal(embedding(ids.int(), w), embedding(ids, w)) and embedding(ids.to(torch.uint8), w).shape == (6, 10, 40)
    out = embedding(ids[:0], w)
    dw, = torch.autograd.grad(out, w, out)
    assert out.shape == (0, 10, 40) and dw.shape == w.shape and float(dw.abs().max()) == 0.0
    assert embedding(ids[0, 0], w).shape == (40,)


def test_gradient_of_the_gradient():
    from hawk_b200 import embedding
    w = torch.randn(6, 4, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 3, 1, 5, 0], device="cuda")
    out = embedding(ids, w, 2.0, padding_idx=0)
    go = torch.randn_like(out).requires_grad_()
    dw, = torch.autograd.grad(out, w, go, create_graph=True)
    u = torch.randn_like(dw)
    dgo, = torch.autograd.grad(dw, go, u)
    want = 2.0 * u[ids]
    want[4] = 0
    assert torch.equal(dgo, want)


def test_refusals():
    from hawk_b200 import embedding
    w, ids = torch.randn(9, 4, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError, match="integers"):
        embedding(ids.float(), w)
    with pytest.raises(ValueError, match="two dimensions"):
        embedding(ids, w[0])
    with pytest.raises(ValueError, match="padding_idx"):
        embedding(ids, w, padding_idx=9)
    with pytest.raises(TypeError, match="float16"):
        embedding(ids, w.half())
    with pytest.raises(RuntimeError, match="cpu"):
        embedding(ids.cpu(), w)


def test_captured_and_other_streams():
    from hawk_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(500, 96, device="cuda")
    ids = _zipf(700, 500, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = embedding(ids, w, 3.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, w[ids] * 3.0)
    from hawk_b200 import ops
    graph = torch.cuda.CUDAGraph()
    go = torch.randn(700, 96, device="cuda")
    with torch.cuda.graph(graph):
        out, dw = embedding(ids, w, 3.0), ops.embedding_bwd(ids, go, 500, 3.0, -1)
    ids.copy_(_zipf(700, 500, g))
    graph.replay()
    assert torch.equal(out, w[ids] * 3.0) and torch.equal(dw, ops.embedding_bwd(ids, go, 500, 3.0, -1))


def test_module_and_model():
    import hawk_b200.model as M
    from hawk_b200 import ops
    torch.manual_seed(0)
    e = M.Embedding(50, 24, padding_idx=3, scale=24 ** 0.5).cuda()
    plain = torch.nn.Embedding(50, 24, padding_idx=3).cuda()
    plain.load_state_dict(e.state_dict())
    ids = torch.randint(0, 50, (5, 9), device="cuda")
    go = torch.randn(5, 9, 24, device="cuda")
    e(ids).backward(go)
    (plain(ids) * 24 ** 0.5).backward(go)
    assert torch.allclose(e.weight.grad, plain.weight.grad, rtol=1e-5, atol=1e-5) and float(e.weight.grad[3].abs().max()) == 0
    model = M.HawkModel(M.HawkConfig(96, 64, 128, 1, 64, 4, 4)).cuda()
    ops.LOG.reset()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        model(ids, ids).backward()
    counts = dict(ops.LOG.counts)
    ops.LOG.enabled = False
    assert counts["embedding_fwd"] == 1 and counts["embedding_bwd"] == 1  # 45 tokens: all in one launch
    cpu = M.Embedding(50, 24, scale=2.0)
    assert torch.equal(cpu(ids.cpu()), 2.0 * cpu.weight[ids.cpu()])
    sparse = M.Embedding(50, 24, sparse=True).cuda()
    sparse(ids).sum().backward()
    assert sparse.weight.grad.is_sparse


@pytest.mark.parametrize("n,V", [(24576, 1), (24577, 1), (60000, 300), (200000, 40)])
def test_runs_longer_than_a_queue(n, V):
    """Blocks whose share is more than their queue holds, and runs of thousands of windows."""
    g = torch.Generator(device="cuda").manual_seed(n)
    _check(_zipf(n, V, g), V, 8, F32)


def test_backward_from_two_threads():
    """Calls whose blocks hold shared memory of different sizes: the kernel's limit belongs to the process."""
    from concurrent.futures import ThreadPoolExecutor

    from hawk_b200 import ops

    def work(n, V):
        with torch.cuda.stream(torch.cuda.Stream()):
            ids, go = torch.arange(n, device="cuda") % V, torch.ones(n, 8, device="cuda")
            for _ in range(300):
                dw = ops.embedding_bwd(ids, go, V, 1.0, -1)
            return bool((dw == (n // V)).all())

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(work, (30000, 64), (5000, 64)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,H", [(1, 524288, 8), (2, 3, 5), (16, 524289, 8), (17, 600000, 8), (256, 511, 130), (257, 512, 64), (1000, 513, 1030),
                                   (2047, 1, 72), (2048, 40, 513), (2049, 40, 513), (2048, 32000, 12), (333, 100000, 2049)])
def test_few_tokens(n, V, H, dtype):
    """Both sides of where one launch serves, all kinds of runs and shares."""
    g = torch.Generator(device="cuda").manual_seed(n + V)
    _check(_zipf(n, V, g), V, H, dtype, scale=0.7)
    ids = torch.randint(0, min(V, 3), (n,), generator=g, device="cuda")
    ids[::5] = V - 1
    _check(ids, V, H, dtype, padding=0 if V > 1 else None)


def test_few_tokens_outside_the_table():
    from hawk_b200 import ops
    ids = torch.tensor([3, -1, 10, 2 ** 40, 9, -2 ** 40, 3], device="cuda")
    go = torch.arange(7.0, device="cuda")[:, None].expand(7, 12).contiguous()
    dw = ops.embedding_bwd(ids, go, 10, 1.0, -1)
    want = torch.zeros(10, 12, device="cuda")
    want[3], want[9] = 6.0, 4.0
    assert torch.equal(dw, want)


def test_module_under_transforms():
    """Forward mode and torch.func see nn.Embedding's own code; the operator itself refuses tangents."""
    import hawk_b200.model as M
    from hawk_b200 import embedding, linear_logprobs, token_logprobs
    from torch.autograd import forward_ad
    from torch.func import functional_call, grad, jacfwd, jacrev, jvp, vmap
    torch.manual_seed(0)
    e = M.Embedding(6, 4, scale=2.0, padding_idx=3).cuda()
    ids = torch.tensor([[1, 5, 3], [0, 1, 1]], device="cuda")
    w, t = e.weight.detach().clone(), torch.randn(6, 4, device="cuda")
    f = lambda w: functional_call(e, {"weight": w}, (ids,))  # noqa: E731
    out, tangent = jvp(f, (w,), (t,))
    assert torch.equal(out, 2 * w[ids]) and torch.equal(tangent, 2 * t[ids])
    with forward_ad.dual_level():
        assert torch.equal(forward_ad.unpack_dual(f(forward_ad.make_dual(w, t))).tangent, 2 * t[ids])
    counts = torch.tensor([1.0, 3.0, 0.0, 0.0, 0.0, 1.0], device="cuda")  # padding has no gradient
    assert torch.equal(grad(lambda w: f(w).sum())(w), 2 * counts[:, None].expand(6, 4))
    jac = torch.zeros(2, 3, 4, 6, 4, device="cuda")
    for i in range(2):
        for k in range(3):
            jac[i, k, range(4), ids[i, k], range(4)] = 2.0
    rev = jac.clone()
    rev[0, 2] = 0.0
    assert torch.equal(jacfwd(f)(w), jac) and torch.equal(jacrev(f)(w), rev)
    both = torch.stack([w, t])
    assert torch.equal(vmap(f)(both), 2 * both[:, ids])
    out = e(ids)  # a batch of upstream gradients for a forward without transforms
    many, = torch.autograd.grad(out, e.weight, torch.stack([torch.ones_like(out), 3 * torch.ones_like(out)]), is_grads_batched=True)
    assert torch.equal(many, torch.stack([k * 2 * counts[:, None].expand(6, 4) for k in (1, 3)]))
    act, head, tokens = torch.randn(3, 8, device="cuda"), torch.randn(5, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for f, x in ((lambda w: embedding(ids, w), w), (lambda a: linear_logprobs(head, a, tokens)[0], act),
                 (lambda x: token_logprobs(x, tokens)[1], act)):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            jvp(f, (x,), (torch.ones_like(x),))
    out = e(ids)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.autograd.grad(out, e.weight, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_module_with_a_table_of_another_kind():
    """A tensor subclass that answers torch's own operators alone, as sharded tables do, keeps them."""
    import hawk_b200.model as M

    class Table(torch.Tensor):
        @staticmethod
        def __new__(cls, data):
            return torch.Tensor._make_wrapper_subclass(cls, data.shape, dtype=data.dtype, device=data.device)

        def __init__(self, data):
            self.data_of = data

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            if func.namespace != "aten":
                raise NotImplementedError(str(func))
            plain = lambda a: a.data_of if isinstance(a, Table) else a  # noqa: E731
            out = func(*(plain(a) for a in args), **{k: plain(a) for k, a in (kwargs or {}).items()})
            return Table(out) if func is torch.ops.aten.detach.default else out

    data, ids = torch.randn(7, 4, device="cuda"), torch.tensor([6, 0, 6], device="cuda")
    e = M.Embedding(7, 4, scale=3.0)
    e.weight = torch.nn.Parameter(Table(data), requires_grad=False)
    assert torch.equal(e(ids), data[ids] * 3.0)
    e.weight = torch.nn.Parameter(data, requires_grad=False)
    assert torch.equal(e(ids.as_subclass(type("Ids", (torch.Tensor,), {}))), data[ids] * 3.0)


def test_gradient_of_the_gradient_outside_the_table():
    """Positions that have no part in the table's gradient have none in its derivative."""
    from hawk_b200 import embedding
    w = torch.randn(6, 4, device="cuda", requires_grad=True)
    ids = torch.tensor([1, -1, 6, 2 ** 40, 5, 0, -6], device="cuda")
    out = embedding(ids, w, 2.0, padding_idx=0)
    go = torch.randn(7, 4, device="cuda").requires_grad_()
    dw, = torch.autograd.grad(out, w, go, create_graph=True)
    u = torch.randn_like(dw)
    dgo, = torch.autograd.grad(dw, go, u)
    want = torch.zeros(7, 4, device="cuda")
    want[0], want[4] = 2.0 * u[1], 2.0 * u[5]
    assert torch.equal(dgo, want)
