"""Views that carry their sign or their zeros beside their memory: the operators read memory."""
import pytest
import torch

from cubutterfly_b200 import torch_ops



def negated(t):
    """The values of `t` (fp32) as a lazily negated view, every second value of its memory."""
    view = torch.complex(torch.ones_like(t), -t).conj().imag
    assert view.is_neg() and torch.equal(view, t)
    return view.requires_grad_(t.requires_grad) if view.is_leaf else view


def test_tensors_of_lazy_zeros_are_refused():
    x, zero = torch.zeros(1, 4, 2, 8), torch._efficientzerotensor((8,))
    for call in (lambda: torch_ops.qk_norm(zero, x), lambda: torch_ops.gated_scan(zero, x, x, x), lambda: torch_ops.block_norm(zero)):
        with pytest.raises(ValueError, match="storage of its own"):
            call()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def same(op, tensors, which):
    """Outputs and gradients of `op` with the tensors `which` as negated views are those with their values."""
    runs = []
    for lazy in (False, True):
        leaves = [t.clone().requires_grad_() for t in tensors]
        # negated twice, once lazily: the leaves' gradients come back through the views
        args = [torch.complex(torch.ones_like(t), -t).conj().imag if lazy and i in which else t for i, t in enumerate(leaves)]
        assert not lazy or all(args[i].is_neg() for i in which)
        outs = op(*args)
        runs.append([*outs, *torch.autograd.grad([o for o in outs], leaves, [normal(90 + i, *o.shape) for i, o in enumerate(outs)])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
def test_negated_gates_of_the_delta_rule(cuda):
    t = [normal(1, 2, 70, 2, 16), torch.nn.functional.normalize(normal(2, 2, 70, 2, 16), dim=-1), normal(3, 2, 70, 4, 8),
         -normal(4, 2, 70, 4).abs(), torch.sigmoid(normal(5, 2, 70, 4)), normal(6, 2, 4, 16, 8)]

    def op(q, k, v, g, beta, state):
        return torch_ops.gated_delta(q, k, v, g, beta, initial_state=state)

    for which in ([3], [4], [3, 4], [0, 1, 2], [5], range(6)):
        same(op, t, which)
    one = [x[..., :1].contiguous() if i < 3 else x for i, x in enumerate(t[:5])]     # one channel: adjacent whatever the stride
    same(torch_ops.gated_delta, one, [0, 1, 2])


@pytest.mark.gpu
def test_negated_views_in_the_other_operators(cuda):
    x, y, w = normal(1, 6, 32), normal(2, 6, 32), normal(3, 32)
    same(lambda x, y, w, p: torch_ops.block_norm(x, y, gate=y * 0.5, pre_weight=w, post_weight=p), [x, y, w, w + 1], range(4))
    s = [normal(i, 2, 20, 8) for i in range(3)] + [normal(7, 8), normal(8, 2, 8)]
    same(lambda x, r, i, d, h: torch_ops.gated_scan(x, r, i, d, initial_state=h), s, range(5))
    same(lambda x, r, i, d: torch_ops.gated_scan(x, r, i, d), [t[..., :1].contiguous() for t in s[:4]], range(4))
    n = [normal(1, 5, 4, 16), normal(2, 5, 2, 16), normal(3, 16), normal(4, 16)]
    same(lambda q, k, a, b: torch_ops.qk_norm(q, k, q_weight=a, k_weight=b), n, range(4))
    positions, frequencies = torch.arange(5, device="cuda"), normal(9, 4).abs()
    want = torch_ops.qk_norm(n[0], n[1], positions=positions, frequencies=frequencies)
    got = torch_ops.qk_norm(n[0], n[1], positions=positions, frequencies=negated(frequencies))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_negated_gradients(cuda):
    """What comes back through a conjugate is negated lazily."""
    q = torch.nn.functional.normalize(normal(1, 1, 70, 2, 16), dim=-1)
    x, w = normal(2, 4, 32), normal(3, 32)

    def through(o, d, lazy):
        if not lazy:
            return (o * d).sum()
        return (torch.complex(torch.zeros_like(o), o).conj() * torch.complex(torch.zeros_like(d), -d)).real.sum().neg()

    ops = [lambda t: torch_ops.gated_delta(t, q, q, q[..., 0] * 0 - 0.1, q[..., 0].abs())[0], lambda t: torch_ops.qk_norm(t, q)[0]]
    for op in ops:
        grads = []
        for lazy in (False, True):
            leaf = q.clone().requires_grad_()
            grads.append(torch.autograd.grad(through(op(leaf), normal(5, *q.shape), lazy), leaf)[0])
        assert torch.allclose(*grads, rtol=1e-6, atol=0)
    # straight into the nodes
    for op, leaf in ((lambda t: torch_ops.block_norm(t, pre_weight=w)[1], x), (ops[0], q), (ops[1], q),
                     (lambda t: torch_ops.gated_scan(t[None], x[None], x[None], w)[0], x)):
        a = leaf.clone().requires_grad_()
        out = op(a)
        d = normal(6, *out.shape)
        (want,) = torch.autograd.grad(out, a, d, retain_graph=True)
        (got,) = torch.autograd.grad(out, a, torch._neg_view(-d))
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_negated_steps_and_pools(cuda):
    q, v, g, beta = normal(1, 3, 2, 16), normal(2, 3, 2, 8), -normal(3, 3, 2).abs(), torch.sigmoid(normal(4, 3, 2))
    pool = normal(5, 3, 2, 16, 8)
    runs = []
    for view in (lambda t: t, negated):
        state = pool.clone()
        runs.append((torch_ops.gated_delta_step(state, view(q), view(q), view(v), view(g), view(beta)), state))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    x, r, decay, rows = normal(6, 3, 8), normal(7, 3, 8), normal(8, 8), normal(9, 3, 8)
    runs = []
    for view in (lambda t: t, negated):
        state = rows.clone()
        runs.append((torch_ops.gated_scan_step(state, view(x), view(r), view(r), view(decay)), state))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    for lazy in (dict(state=torch._neg_view(pool)), dict(state=pool, new_state=torch._neg_view(pool.clone()))):
        with pytest.raises(ValueError, match="lazily negated"):
            torch_ops.gated_delta_step(lazy["state"], q, q, v, g, beta, new_state=lazy.get("new_state"))
    with pytest.raises(ValueError, match="lazily negated"):
        torch_ops.gated_scan_step(torch._neg_view(rows), x, r, r, decay)


@pytest.mark.gpu
def test_transforms_of_lazy_views(cuda):
    x = normal(1, 3, 64)
    assert torch.equal(torch_ops.fwht(torch._neg_view(x)), torch_ops.fwht(-x))
    z = torch.complex(x, normal(2, 3, 64))
    want = torch_ops.fft(z.conj().resolve_conj())
    assert torch.equal(torch_ops.fft(z.conj()), want)
    assert torch.allclose(want, torch.fft.fft(z.conj()), atol=1e-4)
    for out in (torch.empty_like(z).conj(), torch._neg_view(torch.empty_like(z))):
        with pytest.raises(ValueError, match="lazy view"):
            torch_ops.fft(z, out=out)
