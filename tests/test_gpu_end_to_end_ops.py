"""The embedding, the log probabilities, the gradient norm and the clipped update as a user runs them together: a policy-gradient
step of a small model, a padded batch, and scored decoding."""
import math

import pytest
import torch
import torch.utils._python_dispatch

from conftest import rel_l2

pytestmark = pytest.mark.gpu


def _model(seed=0, **kw):
    import hawk_b200.model as M
    torch.manual_seed(seed)
    m = M.HawkModel(M.HawkConfig(96, 64, 128, 2, 64, 4, 4), **kw)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.endswith("resid_proj.weight") or n.endswith("lm_head.weight"):
                p.normal_(0, p.shape[1] ** -0.5)
            elif n.endswith("embed_tokens.weight"):
                p.normal_()
    return m.cuda()


def _plain_scores(logits, tokens):
    logp = torch.log_softmax(logits.double(), -1)
    return logp.gather(-1, tokens[..., None])[..., 0], -(logp.exp() * logp).sum(-1)


def test_scores_follow_the_models_logits():
    """fp32 model: the logits of forward() are fp32 products of fp32 activations, those of token_logprobs bf16 products: operands
    rounded by 2^-9 each over sums of 64 products, logits of about 1 to 4: under 3e-2."""
    m = _model()
    ids = torch.randint(1, 96, (3, 41), device="cuda")
    with torch.no_grad():
        lp, H = m.token_logprobs(ids)
        rlp, rH = _plain_scores(m(ids)[:, :-1], ids[:, 1:])
    assert lp.shape == H.shape == (3, 40)
    assert float((lp - rlp).abs().max()) <= 3e-2 and float((H - rH).abs().max()) <= 3e-2
    # and its mean is the training loss up to the rounding of the logits to bf16
    with torch.no_grad():
        assert abs(float(m(ids, ids)) + float(lp.mean())) <= 1e-2


def test_policy_gradient_step():
    """Embedding -> layers -> log probabilities with an entropy bonus -> backward -> clip -> AdamW, against autograd through the
    model's own logits in the same precision of the trunk; gradients to the bf16 bound of the head's products (2e-2, the bound of
    the model's other gradients)."""
    from hawk_b200.train import FusedAdamW, clip_grad_norm_
    m, ref = _model(1), _model(1)
    ids = torch.randint(1, 96, (4, 33), device="cuda")
    labels = ids.clone()
    labels[1, 20:] = -1           # a shorter sequence
    labels[3, :] = -100           # and one of nothing but padding
    adv = torch.randn(4, 32, device="cuda")
    lp, H = m.token_logprobs(ids, labels)
    loss = -(adv * lp).sum() / 60 - 0.01 * H.sum() / 60
    loss.backward()
    named = labels[:, 1:] >= 0
    rlp, rH = _plain_scores(ref(ids)[:, :-1], ids[:, 1:])
    rloss = -(adv.double() * rlp * named).sum() / 60 - 0.01 * (rH * named).sum() / 60
    rloss.backward()
    assert float(lp[3].abs().max()) == 0 and float(H[1, 19:].abs().max()) == 0
    assert abs(float(loss) - float(rloss)) <= 2e-2 * abs(float(rloss))
    for (n, p), q in zip(m.named_parameters(), ref.parameters()):
        assert rel_l2(p.grad, q.grad) <= 2e-2, n
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in m.parameters()))
    opt = FusedAdamW(m.parameters(), lr=1e-3, max_grad_norm=0.1 * norm)
    other = _model(1)
    for p, q in zip(other.parameters(), m.parameters()):
        p.grad = q.grad.clone()
    opt.step()
    got = clip_grad_norm_(other.parameters(), 0.1 * norm)
    FusedAdamW(other.parameters(), lr=1e-3).step()
    assert abs(float(opt.grad_norm) - norm) <= 1e-6 * norm and float(got) == float(opt.grad_norm)
    for (n, p), q in zip(m.named_parameters(), other.named_parameters()):
        assert rel_l2(p, q[1]) <= 1e-6, n  # clip, then update, is the update that clips


def test_padding_does_not_reach_the_gradients():
    """Positions behind the last named label change nothing: the recurrence is causal, and their rows are left out."""
    m = _model(2)
    ids = torch.randint(1, 96, (2, 30), device="cuda")
    labels = ids.clone()
    labels[:, 18:] = -1

    def grads(x):
        m.zero_grad(set_to_none=True)
        lp, H = m.token_logprobs(x, labels)
        (lp.sum() + H.sum()).backward()
        return lp.detach(), [p.grad.clone() for n, p in m.named_parameters() if not n.startswith("embed")]
    lp, g = grads(ids)
    other = ids.clone()
    other[:, 18:] = torch.randint(1, 96, (2, 12), device="cuda")
    lp2, g2 = grads(other)
    assert torch.equal(lp, lp2)
    for a, b in zip(g, g2):  # sums over rows whose gradient is zero in both: the same terms
        assert rel_l2(a, b) <= 1e-6


def test_autocast_training_step_with_everything():
    from hawk_b200 import ops
    from hawk_b200.train import Trainer
    import hawk_b200.model as M
    tr = Trainer(M.HawkConfig(96, 64, 128, 2, 64, 4, 4), "cuda", seed=1, max_grad_norm=1.0)
    ids = torch.randint(1, 96, (2, 33), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        lp, H = tr.model.token_logprobs(ids)
    (-lp.mean()).backward()
    g1 = [p.grad.clone() if p.grad is not None else None for p in tr.model.parameters()]
    tr.model.zero_grad(set_to_none=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        tr.model(ids, ids).backward()
    for a, p in zip(g1, tr.model.parameters()):  # minus the mean log probability is the training loss
        if float(p.grad.abs().max()) > 0:
            assert rel_l2(a, p.grad) <= 3e-2
    ops.LOG.reset()
    tr.step(ids)
    counts = dict(ops.LOG.counts)
    ops.LOG.enabled = False
    assert counts["grad_norm"] == 2 and counts["embedding_bwd"] == 1 and math.isfinite(float(tr.grad_norm))


@pytest.mark.parametrize("use_graph", [False, True])
def test_scored_decoding(use_graph):
    from hawk_b200.generate import GraphedDecoder
    m = _model(3, use_cache=True).bfloat16()
    dec = GraphedDecoder(m, 5, autocast=False, use_graph=use_graph)
    with pytest.raises(AssertionError, match="prefill"):
        dec.logprobs(torch.zeros(5, dtype=torch.int64, device="cuda"))
    logits = dec.prefill(torch.randint(1, 96, (5, 9), device="cuda"))
    for _ in range(3):
        last = logits[:, -1].float()
        chosen = last.argmax(-1)
        chosen[2] = -1  # a sequence that has ended
        lp, H, best, ids = dec.logprobs(chosen, 3)
        rlp, rH = _plain_scores(last, chosen.clamp(min=0))
        live = torch.tensor([0, 1, 3, 4], device="cuda")
        assert float((lp - rlp)[live].abs().max()) <= 1e-5 and float((H - rH)[live].abs().max()) <= 1e-4
        assert torch.equal(ids[live, 0], chosen[live]) and torch.equal(best[live, 0], lp[live])
        assert float(lp[2]) == 0 and ids[2].tolist() == [-1] * 3
        logits = dec.step(chosen.clamp(min=0)[:, None])
        assert torch.equal(dec.logprobs(chosen[:, None])[0], dec.logprobs(chosen)[0])


def test_a_cached_model_refuses_whole_sequences():
    with pytest.raises(ValueError, match="use_cache"):
        _model(4, use_cache=True).token_logprobs(torch.zeros(1, 4, dtype=torch.int64, device="cuda"))


def test_through_the_dispatcher():
    """The same calls where torch has to see the operators: under modes, and as torch.library's checks want them."""
    import hawk_b200 as h
    from hawk_b200 import ops

    class Passes(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Dispatches(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(50, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    a = torch.randn(3, 7, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    x = torch.randn(3, 7, 50, generator=g, device="cuda").requires_grad_()
    ids = torch.randint(-1, 50, (3, 7), generator=g, device="cuda")

    def everything():
        out = [h.embedding(ids.clamp(min=0), w, 2.0, 3), *h.linear_logprobs(w, a, ids), *h.token_logprobs(x, ids, 4)]
        grads = torch.autograd.grad([o.float().sum() for o in out if o.requires_grad], [w, a, x])
        return [*out, *grads]
    direct = everything()
    for context in (Passes, Dispatches):
        with context():
            seen = everything()
        assert all(torch.equal(p, q) for p, q in zip(direct, seen))
    tests = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_static")
    torch.library.opcheck(ops.embedding_fwd, (ids.clamp(min=0), w, 2.0, 3), test_utils=tests)
    torch.library.opcheck(ops.token_logprobs_fwd, (x, ids, 4), test_utils=tests)
    torch.library.opcheck(ops.linear_logprobs_fwd, (w.detach(), a.detach(), ids, False), test_utils=tests[:1] + tests[2:3])


def test_saved_bytes_are_what_the_fake_says():
    from hawk_b200 import ops
    from torch._subclasses.fake_tensor import FakeTensorMode
    for wdt, adt, V, N, H in [(torch.float32, torch.float32, 300, 5, 64), (torch.bfloat16, torch.bfloat16, 129, 70, 8),
                              (torch.bfloat16, torch.float32, 1000, 33, 24)]:
        for grad in (False, True):
            args = (torch.zeros(V, H, dtype=wdt, device="cuda"), torch.zeros(N, H, dtype=adt, device="cuda"),
                    torch.zeros(N, dtype=torch.int64, device="cuda"))
            real = ops.linear_logprobs_fwd(*args, grad)
            with FakeTensorMode() as mode:
                fake = ops.linear_logprobs_fwd(*(mode.from_tensor(a) for a in args), grad)
            assert [t.shape for t in real] == [t.shape for t in fake] and [t.dtype for t in real] == [t.dtype for t in fake]


def test_a_first_call_inside_a_capture():
    """The status word of the tensor-core kernels made while capturing belongs to the graph: eager calls before its first replay
    must not read it."""
    from hawk_b200 import linear_logprobs, ops
    g = torch.Generator(device="cuda").manual_seed(0)
    w, a = (torch.randn(200, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    t = torch.randint(0, 200, (200,), generator=g, device="cuda")
    want = linear_logprobs(w, a, t)
    kept = dict(ops._ce_status)
    torch.cuda.synchronize()
    ops._ce_status.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear_logprobs(w, a, t)
        assert not ops._ce_status
        assert all(torch.equal(x, y) for x, y in zip(linear_logprobs(w, a, t), want))
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        ops.check_device_status()
    finally:
        ops._ce_status.update(kept)


def test_prompt_logits_are_not_kept():
    from hawk_b200.generate import GraphedDecoder
    m = _model(5, use_cache=True).bfloat16()
    dec = GraphedDecoder(m, 2, autocast=False, use_graph=False)
    logits = dec.prefill(torch.randint(1, 96, (2, 50), device="cuda"))
    assert dec._latest.untyped_storage().nbytes() == logits[:, -1].numel() * logits.element_size()
    assert torch.equal(dec._latest[:, 0], logits[:, -1])


def test_two_calls_at_once_on_two_streams():
    """Nothing is shared between calls but the status word."""
    from hawk_b200 import embedding, grad_norm, linear_logprobs, ops, token_logprobs
    g = torch.Generator(device="cuda").manual_seed(3)
    sets = []
    for k in range(2):
        w = torch.randn(3000, 128, generator=g, device="cuda").bfloat16()
        a = torch.randn(700, 128, generator=g, device="cuda").bfloat16()
        t = torch.randint(0, 3000, (700,), generator=g, device="cuda")
        sets.append((w, a, t, torch.randn(700, 3000, generator=g, device="cuda")))

    def run(w, a, t, x):
        lp, H, saved = ops.linear_logprobs_fwd(w, a, t, True)
        return [lp, H, *ops.linear_logprobs_bwd(w, a, t, saved, lp, H, lp, H, True, True), *token_logprobs(x, t, 7), embedding(t, w, 2.0),
                ops.embedding_bwd(t, a, 3000, 1.0, -1), grad_norm([w, a, x])]
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(run(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(out, want[k]))


def test_batched_by_vmap():
    from hawk_b200 import embedding, linear_logprobs, token_logprobs
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(-1, 9, (4, 5), generator=g, device="cuda")
    w, x, a = (torch.randn(s, generator=g, device="cuda") for s in ((9, 8), (4, 5, 9), (4, 5, 8)))
    known = ids.clamp(min=0)
    assert torch.equal(torch.vmap(lambda i: embedding(i, w, 2.0))(known), 2.0 * w[known])
    assert torch.equal(torch.vmap(lambda v: embedding(known, v))(torch.stack([w, -w])), torch.stack([w[known], -w[known]]))
    for f, args in ((lambda x, t: token_logprobs(x, t, 2), (x, ids)), (token_logprobs, (x, ids)),
                    (lambda a, t: linear_logprobs(w, a, t), (a, ids))):
        assert all(torch.equal(p, q) for p, q in zip(torch.vmap(f)(*args), f(*args)))


@pytest.mark.parametrize("op", ["token_logprobs", "linear_logprobs", "embedding"])
def test_compiled_gradients_are_the_eager_ones(op):
    import hawk_b200
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 300, (4, 50), generator=g, device="cuda")
    w, x, a = (torch.randn(s, generator=g, device="cuda", requires_grad=True) for s in ((300, 64), (4, 50, 300), (4, 50, 64)))
    f, leaves = {"token_logprobs": (lambda: sum(hawk_b200.token_logprobs(x, ids - 3)[:2]), (x,)),
                 "linear_logprobs": (lambda: sum(hawk_b200.linear_logprobs(w, a, ids - 3)), (w, a)),
                 "embedding": (lambda: hawk_b200.embedding(ids, w, 3.0, 7) * a, (w, a))}[op]
    results = []
    for call in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        out = call()
        results.append([out, *torch.autograd.grad(out, leaves, torch.cos(torch.arange(out.numel(), device="cuda").view(out.shape)))])
    assert all(torch.equal(p, q) for p, q in zip(*results))
