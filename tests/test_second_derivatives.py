"""Gradients of gradients: the backward kernels have none, and asking for one is an error, not a missing term.

The kernels are stood in for by torch code whose results carry no graph, as those of the C ABI calls do, so
this runs without a GPU."""
import importlib

import pytest

torch = pytest.importorskip("torch")

fa = importlib.import_module("tf-custom-flash-attention_b200")


def norm(x, w, eps):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


@pytest.fixture
def rope_on_cpu(monkeypatch):
    def forward(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved):
        return norm(q, q_weight, eps), norm(k, k_weight, eps)

    def backward(q, k, dq_out, dk_out, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved):
        leaves = [None if x is None else x.detach().requires_grad_() for x in (q, k, q_weight, k_weight)]
        with torch.enable_grad():
            outs = forward(leaves[0], leaves[1], leaves[2], leaves[3], table, q_positions, k_positions, eps, interleaved)
        got = iter(torch.autograd.grad(outs, [x for x in leaves if x is not None], (dq_out.detach(), dk_out.detach())))
        return tuple(None if x is None else next(got) for x in leaves)

    monkeypatch.setattr(fa.rotary, "qk_norm_rope", forward)
    monkeypatch.setattr(fa.rotary, "qk_norm_rope_grad", backward)


def rope_loss(x, square):
    a, b = fa.autograd.qk_norm_rope(x, 2 * x, torch.ones(8), None)
    y = (a + b.flip(1)) * torch.linspace(-1, 1, 8)
    return (y * y).sum() if square else y.sum()


def project(seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(8, 8, generator=g).requires_grad_(), torch.randn(1, 5, 2, 8, generator=g)


@pytest.mark.parametrize("square", [True, False])  # the gradient of the results depends on the leaf, or does not
def test_rope_second_derivative_is_refused(rope_on_cpu, square):
    w, x = project()
    h = (x @ w).tanh()
    (g,) = torch.autograd.grad(rope_loss(h, square), w, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad((g * g).sum(), w)


def test_rope_first_derivative_is_the_same_with_a_graph(rope_on_cpu):
    w, x = project()
    (a,) = torch.autograd.grad(rope_loss((x @ w).tanh(), True), w)
    (b,) = torch.autograd.grad(rope_loss((x @ w).tanh(), True), w, create_graph=True)
    assert torch.equal(a, b)


def test_rope_terms_beside_it_keep_their_second_derivative(rope_on_cpu):
    """A penalty on a gradient that does not pass the operator is differentiated as before."""
    w, x = project()
    u = torch.randn(8, generator=torch.Generator().manual_seed(5)).requires_grad_()
    loss = rope_loss((x @ w).tanh(), True) + (u ** 3).sum()
    gu, _ = torch.autograd.grad(loss, (u, w), create_graph=True)
    (second,) = torch.autograd.grad(gu.sum(), u)
    assert torch.allclose(second, 6 * u)


def attend(q, k, v, scale):
    s = q @ k.transpose(-1, -2) * scale
    return s.softmax(-1) @ v, s.logsumexp(-1)


@pytest.fixture
def sdpa_on_cpu(monkeypatch):
    def forward(q, k, v, seed, offset, *, scale, dropout, causal_mask):
        return attend(q, k, v, scale)

    def backward(q, k, v, o, stats, d_o, seed, offset, *, dropout, scale, causal_mask, d_stats=None):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        with torch.enable_grad():
            o, s = attend(*leaves, scale)
        return torch.autograd.grad((o, s), leaves, (d_o.detach(), torch.zeros_like(s) if d_stats is None else d_stats.detach()))

    monkeypatch.setattr(fa.ops, "sdpa", forward)
    monkeypatch.setattr(fa.ops, "sdpa_grad", backward)
    monkeypatch.setattr(fa.ops, "sdpa_bshd", lambda *a, **kw: forward(*a, **kw))
    monkeypatch.setattr(fa.ops, "sdpa_grad_bshd", lambda *a, **kw: backward(*a, **kw))


def with_stats(h, differentiable):
    o, s = fa.autograd.sdpa_with_stats(h, 2 * h, h, 0, 0, differentiable_stats=differentiable)
    return o * s.detach()[..., None] + (s[..., None] if differentiable else 0)


ATTENTIONS = [lambda h: fa.autograd.sdpa(h, 2 * h, h, 0, 0), lambda h: fa.autograd.sdpa_bshd(h, h, h, 0, 0),
              lambda h: with_stats(h, False), lambda h: with_stats(h, True)]


@pytest.mark.parametrize("op", range(4))
@pytest.mark.parametrize("square", [True, False])
def test_attention_second_derivative_is_refused(sdpa_on_cpu, op, square):
    w, x = project()
    out = ATTENTIONS[op]((x[0] @ w).tanh())
    loss = (out * out).sum() if square else out.sum()
    (first,) = torch.autograd.grad(loss, w, retain_graph=True)
    (g,) = torch.autograd.grad(loss, w, create_graph=True)
    assert torch.equal(first, g)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad((g * g).sum(), w)
