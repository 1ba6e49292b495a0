"""The gradient through ops.moe_route and the torch operator, on the CPU: the oracle stands in for the kernels for
the duration of a test."""

import itertools

import numpy as np
import pytest
import torch

import mosaicist_b200.torch_ops as O
from mosaicist_b200 import ops
from oracle import route as R


@pytest.fixture()
def calls():
    seen = []

    def forward(logits, topk, score, bias, groups, topk_groups, group_top, renormalize, scale):
        ids, w = R.route(logits.numpy(), topk, score, None if bias is None else bias.numpy(), groups, topk_groups, group_top, renormalize, scale)
        return torch.from_numpy(ids), torch.from_numpy(w.astype(np.float32))

    def backward(grad, logits, ids, weights, score, renormalize, scale):
        assert grad.is_contiguous() and grad.dtype == torch.float32
        seen.append((score, renormalize, scale))
        got = R.route_backward(*(t.detach().numpy() for t in (grad, logits, ids, weights)), score, renormalize, scale)
        return torch.from_numpy(got).to(logits.dtype)

    lib = torch.library.Library("mosaicist_sm100a", "IMPL")
    lib.impl("moe_route", forward, "CPU")
    lib.impl("moe_route_backward", backward, "CPU")
    yield seen
    lib._destroy()


CASES = list(itertools.product(["softmax", "sigmoid"], [True, False], [False, True]))


@pytest.mark.parametrize("score,renormalize,biased", CASES)
def test_gradient_of_the_logits(calls, score, renormalize, biased):
    """Against central differences of the weights in 64 bits, the choice held."""
    rng = np.random.default_rng(0)
    T, E, k, scale, h = 6, 16, 4, 2.5, 1e-5
    x = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)).requires_grad_()
    bias = torch.from_numpy((rng.standard_normal(E) * 0.1).astype(np.float32)).requires_grad_() if biased else None
    g = torch.from_numpy(rng.standard_normal((T, k)).astype(np.float32))
    ids, w = ops.moe_route(x, k, score, bias, 4, 2, 2, renormalize, scale)
    assert w.requires_grad and not ids.requires_grad
    got = torch.autograd.grad((w * g).sum(), x)[0].numpy()
    assert calls == [(score, renormalize, scale)] and (bias is None or bias.grad is None)
    x64, i = x.detach().numpy().astype(np.float64), ids.numpy()
    for e in range(E):
        d = np.zeros((T, E))
        d[:, e] = h
        diff = (R.weights_of(x64 + d, i, score, renormalize, scale) - R.weights_of(x64 - d, i, score, renormalize, scale)) / (2 * h)
        # h^2 / 6 of the third derivative (below 1), the differences' own cancellation (2^-52 / h, four terms) and
        # fp32's share of weights and result
        off = 4 * scale * float(g.abs().max()) * (h * h + 2.0 ** -52 / h + 8 * 2.0 ** -24)
        assert np.abs(got[:, e] - (g.numpy() * diff).sum(1)).max() <= off


def test_a_step_of_a_router(calls):
    """Through what makes the logits and what uses the weights, an expanded gradient among them; twice."""
    x, wr = torch.randn(5, 8), torch.randn(12, 8, requires_grad=True)
    for _ in range(2):
        ids, w = O.moe_route(x @ wr.t(), 3, "sigmoid", None, 1, 1, 1, True, 1.0)
        (w.sum(dim=1) * torch.arange(5.0)).sum().backward()
    assert wr.grad.shape == wr.shape and len(calls) == 2
    # renormalised weights add up to 1 whatever the logits are
    assert float(wr.grad.abs().max()) <= 64 * 2.0 ** -24 * float(x.abs().max())
    w = O.moe_route(x @ wr.t(), 3, "softmax", None, 1, 1, 1, False, 2.0)[1]
    wr.grad = None
    w[:, 0].sum().backward()
    assert float(wr.grad.abs().max()) > 0


def test_arguments_as_the_plain_path_takes_them(calls):
    x = torch.randn(5, 8, requires_grad=True)
    want = ops.moe_route(x, 2, groups=4, topk_groups=2, renormalize=True, scale=2.0)
    got = ops.moe_route(x, np.int64(2), groups=np.int32(4), topk_groups=np.int64(2), renormalize=1, scale=2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for kw in (dict(topk=2.0), dict(topk=2, groups=4.0), dict(topk=2, scale="x")):
        with pytest.raises((TypeError, ValueError)):
            ops.moe_route(x, **kw)


def test_where_no_gradient_is_asked_for(calls):
    x = torch.randn(5, 8, requires_grad=True)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):      # the plain path, which has no stand-in
        ops.moe_route(x, 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.moe_route(x, 2, out=(torch.zeros(5, 2, dtype=torch.int32), torch.zeros(5, 2)))
    with pytest.raises(ValueError, match="score"):
        ops.moe_route(x, 2, score="tanh")
    w = ops.moe_route(x, 2)[1]
    with pytest.raises(RuntimeError, match="not implemented|no autograd formula"):   # no second derivative
        g = torch.autograd.grad(w[:, 0].sum(), x, create_graph=True)[0]
        torch.autograd.grad(g.sum(), x)
