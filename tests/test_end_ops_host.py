"""Argument checks of the embedding, log-probability and gradient-norm entry points; no GPU needed."""
import ctypes
import struct

import pytest
import torch

import hawk_b200._lib as L


def _table(*rows):
    return struct.pack(f"{3 * len(rows)}q", *(v for r in rows for v in r))


def test_grad_norm_argument_validation():
    lib = L.load()
    p = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
    good = _table((4096, 8, 0))
    ws = lib.hawk_grad_norm_workspace_bytes(1)
    assert lib.hawk_grad_norm(None, 1, 1.0, p, p, ws, None) == -1
    assert lib.hawk_grad_norm(good, 1, 1.0, None, p, ws, None) == -1
    assert lib.hawk_grad_norm(good, 0, 1.0, p, p, ws, None) == -2
    assert lib.hawk_grad_norm(good, 1, -1.0, p, p, ws, None) == -2
    assert lib.hawk_grad_norm(good, 1, float("nan"), p, p, ws, None) == -2
    assert lib.hawk_grad_norm(good, 1, 1.0, p, None, ws, None) == -5
    assert lib.hawk_grad_norm(good, 1, 1.0, p, p, ws - 1, None) == -5
    assert lib.hawk_grad_norm(good, 1, 1.0, p, ctypes.c_void_p(4100), ws, None) == -4
    for row, code in [((0, 8, 0), -1), ((4096, 0, 0), -2), ((4096, 8, 2), -3), ((4098, 8, 0), -4), ((4097, 8, 1), -4),
                      ((4096, 1 << 41, 0), -2)]:
        assert lib.hawk_grad_norm(_table(row), 1, 1.0, p, p, ws, None) == code
        assert lib.hawk_scale_multi(_table(row), 1, p, None) == code
    assert lib.hawk_grad_norm(_table(*[(4096, 1 << 40, 0)] * 64), 64, 1.0, p, p, ws, None) == -2  # beyond 32 bits of chunks
    assert lib.hawk_scale_multi(good, 1, None, None) == -1
    assert lib.hawk_scale_multi(good, 1, ctypes.c_void_p(4098), None) == -4
    assert lib.hawk_grad_norm_workspace_bytes(1025) == 2 * lib.hawk_grad_norm_workspace_bytes(1024)
    adam = (1e-3, 0.9, 0.999, 1e-8, 0.1)
    one = struct.pack("6Q", 4096, 4096, 4096, 4096, 0, 8)
    assert lib.hawk_adamw_multi_scaled(one, 1, *adam, 1, ctypes.c_void_p(4098), None) == -4


def test_norm_refuses_cpu_tensors():
    from hawk_b200 import grad_norm
    with pytest.raises(RuntimeError, match="CUDA"):
        grad_norm([torch.ones(3)])


def test_cpu_trainer_clips():
    """The plumbing of max_grad_norm where the trainer runs torch's own optimiser (no kernels on the CPU)."""
    from hawk_b200.train import Trainer
    tr = Trainer.__new__(Trainer)
    tr.model = torch.nn.Linear(4, 3)
    tr.opt = torch.optim.SGD(tr.model.parameters(), lr=1.0)
    tr.max_grad_norm, tr.grad_norm = 0.5, None
    before = [p.detach().clone() for p in tr.model.parameters()]
    for p in tr.model.parameters():
        p.grad = torch.ones_like(p)
    tr._update()
    assert abs(float(tr.grad_norm) - 15 ** 0.5) < 1e-6
    moved = torch.cat([(b - p.detach()).view(-1) for b, p in zip(before, tr.model.parameters())])
    assert abs(float(moved.norm()) - 0.5) < 1e-5 and all(p.grad is None for p in tr.model.parameters())


def test_embedding_argument_validation():
    lib = L.load()
    p = ctypes.c_void_p(4096)
    assert lib.hawk_embedding_fwd(None, p, p, 4, 10, 8, 1.0, 0, None) == -1
    assert lib.hawk_embedding_fwd(p, p, p, 0, 10, 8, 1.0, 0, None) == -2
    assert lib.hawk_embedding_fwd(p, p, p, 4, 10, 0, 1.0, 0, None) == -2
    assert lib.hawk_embedding_fwd(p, p, p, 4, 1 << 31, 8, 1.0, 0, None) == -2
    assert lib.hawk_embedding_fwd(p, p, p, 1 << 31, 10, 8, 1.0, 0, None) == -2
    assert lib.hawk_embedding_fwd(p, p, p, 4, 10, 8, 1.0, 5, None) == -3
    assert lib.hawk_embedding_fwd(p, ctypes.c_void_p(4098), p, 4, 10, 8, 1.0, 0, None) == -4
    ws = lib.hawk_embedding_bwd_workspace_bytes(5000, 10, 8)
    assert ws >= 100 * 4 + 11 * 4 + 3 * 8 * 4
    assert lib.hawk_embedding_bwd(p, p, p, None, ws, 5000, 10, 8, -1, 1.0, 0, None) == -5
    assert lib.hawk_embedding_bwd(p, p, p, p, ws - 1, 5000, 10, 8, -1, 1.0, 0, None) == -5
    assert lib.hawk_embedding_bwd(p, p, p, ctypes.c_void_p(4100), ws, 100, 10, 8, -1, 1.0, 0, None) == -4
    assert lib.hawk_embedding_bwd(p, None, p, p, ws, 100, 10, 8, -1, 1.0, 0, None) == -1
    assert lib.hawk_embedding_bwd_workspace_bytes(2048, 1 << 19, 8) == 0 < lib.hawk_embedding_bwd_workspace_bytes(2048, (1 << 19) + 1, 8)
    assert [lib.hawk_embedding_bwd_kernels(*a) for a in ((2048, 10, 8), (2049, 10, 8), (16, 1 << 20, 8), (17, 1 << 20, 8))] == [1, 3, 2, 3]


def test_embedding_refuses_cpu_tensors():
    from hawk_b200 import embedding
    with pytest.raises(RuntimeError, match="CUDA"):
        embedding(torch.zeros(3, dtype=torch.int64), torch.ones(4, 8))
    with pytest.raises(TypeError, match="integers"):
        embedding(torch.zeros(3), torch.ones(4, 8))


def test_token_logprobs_argument_validation():
    lib = L.load()
    p = ctypes.c_void_p(4096)
    call = lambda x=p, ld=10, rows=4, V=10, top=3, best=p, dt=0: lib.hawk_token_logprobs(  # noqa: E731
        x, ld, p, p, p, p, best, best, rows, V, top, dt, None)
    assert call(x=None) == -1 and call(best=None) == -1
    assert call(rows=0) == call(V=0, top=0) == call(ld=9) == call(top=11) == call(top=-1) == call(V=64, ld=64, top=33) == -2
    assert call(rows=1 << 28) == call(V=1 << 28, ld=1 << 28) == -2
    assert call(dt=3) == -3 and call(x=ctypes.c_void_p(4098)) == -4
    back = lambda x=p, ld=10, rows=4, dx=p, dt=1: lib.hawk_token_logprobs_bwd(  # noqa: E731
        x, ld, p, p, p, p, None, None, dx, rows, 10, dt, None)
    assert back(x=None) == back(dx=None) == -1
    assert back(ld=9) == back(rows=0) == -2 and back(dt=2) == -3 and back(dx=ctypes.c_void_p(4097)) == -4


def test_token_logprobs_refuses_cpu_tensors():
    from hawk_b200 import token_logprobs
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="top"):
        token_logprobs(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 9)


def test_linear_logprobs_argument_validation():
    lib = L.load()
    p = ctypes.c_void_p(4096)
    saved = lib.hawk_linear_logprobs_saved_bytes(4, 64, 300, 0, 1, 1)
    assert saved >= 300 * 64 * 2 + 4 * 304 * 2 + 4 * 3 * 16 and lib.hawk_linear_logprobs_saved_bytes(4, 64, 300, 1, 1, 0) < saved
    fwd = lambda w=p, sv=p, n=saved, N=4, H=64, dt=0, st=p: lib.hawk_linear_logprobs(  # noqa: E731
        w, p, p, p, p, sv, n, N, H, 300, dt, 1, 1, st, None)
    assert fwd(w=None) == fwd(st=None) == -1 and fwd(N=0) == fwd(H=60) == -2 and fwd(dt=4) == -3
    assert fwd(sv=None) == fwd(n=saved - 1) == -5 and fwd(w=ctypes.c_void_p(4104)) == -4
    scratch = lib.hawk_linear_logprobs_scratch_bytes(4, 64, 300, 1, 1, 1)
    bwd = lambda dw=p, sc=p, n=scratch, sv=saved, H=64: lib.hawk_linear_logprobs_bwd(  # noqa: E731
        p, p, p, p, sv, p, p, None, None, dw, 0, None, 0, sc, n, 4, H, 300, 0, 1, p, None)
    assert bwd(dw=None) == -1 and bwd(H=4) == -2 and bwd(sc=None) == bwd(sv=saved - 1) == -5 and bwd(dw=ctypes.c_void_p(4100)) == -4
    need = lib.hawk_linear_logprobs_scratch_bytes(4, 64, 300, 1, 1, 0)
    assert bwd(n=need - 1) == -5
    assert lib.hawk_linear_logprobs_kernels(4, 64, 300, 0, 1, 0, 0) == 3


def test_linear_logprobs_refuses_cpu_tensors():
    from hawk_b200 import linear_logprobs
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_logprobs(torch.zeros(9, 8), torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64))


# what may ask for a forward-mode derivative, each the derivative of f at x in the direction t
def _dual(f, x, t):
    with torch.autograd.forward_ad.dual_level():
        return torch.autograd.forward_ad.unpack_dual(f(torch.autograd.forward_ad.make_dual(x, t))).tangent


FORWARD_MODE = [_dual, lambda f, x, t: torch.func.jvp(f, (x,), (t,))[1], lambda f, x, t: torch.func.jacfwd(f)(x),
                lambda f, x, t: torch.func.jvp(torch.func.vmap(f), (x,), (t,)), lambda f, x, t: torch.func.jvp(lambda a: f(x=a), (x,), (t,)),
                lambda f, x, t: torch.func.jvp(lambda a: torch.func.jvp(f, (a,), (t,))[1], (x,), (t,))]


@pytest.mark.parametrize("way", range(len(FORWARD_MODE)))
def test_operators_without_a_forward_derivative_refuse_tangents(way):
    """Operators of the form of the embedding and the log probabilities: the dispatcher would answer with a tangent of zeros."""
    from hawk_b200 import ops

    @ops._operator(f"hawk_b200_test::reverse_only_{way}", mutates_args=(), reverse_only=True)
    def op(x: torch.Tensor) -> torch.Tensor:
        return 2 * x
    op.register_autograd(lambda ctx, g: 2 * g, setup_context=lambda ctx, inputs, output: None)
    x, t = torch.ones(3, 2), torch.ones(3, 2)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        FORWARD_MODE[way](op, x, t)
    assert torch.equal(torch.func.vmap(op)(x), 2 * x)  # other transforms are answered as before
    with torch.autograd.forward_ad.dual_level():
        assert torch.equal(op(x), 2 * x)  # no tangent
    assert all(o.reverse_only for o in (ops.embedding_fwd, ops.embedding_bwd, ops.token_logprobs_fwd, ops.token_logprobs_bwd,
                                        ops.linear_logprobs_fwd, ops.linear_logprobs_bwd))


def test_embedding_takes_its_argument_by_name():
    """The model's table is called as nn.Embedding is."""
    import inspect

    import hawk_b200.model as M
    e, ids = M.HawkModel(M.HawkConfig(96, 64, 128, 1, 64, 4, 4)).embed_tokens, torch.tensor([3, 95])
    assert torch.equal(e(input=ids), e.weight[ids])
    assert inspect.signature(type(e).forward).parameters.keys() == inspect.signature(torch.nn.Embedding.forward).parameters.keys()
