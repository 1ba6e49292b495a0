"""Expert routing (ops.moe_route, ops.moe_route_backward) against the oracle in 64 bits."""

import itertools

import numpy as np
import pytest
import torch

from oracle import route as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# Weights: expf is off by at most 2 ulp (2^-22), each of the other roundings by 2^-24: the chosen scores'
# sum (up to five additions over lanes), two quotients, the scale.  A softmax that is not renormalised
# divides by a sum of terms that are off by 2^-22 + |x - max| 2^-24 (|x - max| < 20 here matters: e^-20
# of the largest), and up to 37 additions.
W_TOL = 2.0 ** -22 * 2 + 10 * 2.0 ** -24
W_TOL_SUM = 2.0 ** -22 * 2 + (20 + 37 + 10) * 2.0 ** -24


def _run(logits, topk, dtype="f32", bias=None, **kw):
    from mosaicist_b200 import ops

    x = torch.from_numpy(logits.astype(np.float32)).to(DT[dtype]).cuda()
    b = None if bias is None else torch.from_numpy(bias.astype(np.float32)).cuda()
    ids, w = ops.moe_route(x, topk, bias=b, **kw)
    seen = x.float().cpu().numpy()
    return seen, ids, w


def _check(logits, topk, dtype="f32", bias=None, score="softmax", renormalize=True, **kw):
    seen, ids, w = _run(logits, topk, dtype, bias, score=score, renormalize=renormalize, **kw)
    want_ids, want_w = R.route(seen, topk, score, None if bias is None else bias.astype(np.float32), renormalize=renormalize, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    tol = W_TOL_SUM if score == "softmax" and not renormalize else W_TOL
    # (an absolute 2^-126: e^x below that is flushed to zero)
    assert (np.abs(w.cpu().numpy() - want_w) <= tol * want_w + 2.0 ** -126 * kw.get("scale", 1.0)).all()
    return seen, ids, w


SHAPES = [  # experts, topk, groups, topk_groups, group_top
    (1, 1, 1, 1, 1), (2, 1, 1, 1, 1), (31, 5, 1, 1, 1), (61, 4, 1, 1, 1), (64, 32, 1, 1, 1), (160, 6, 8, 3, 1),
    (160, 6, 8, 3, 2), (256, 8, 8, 4, 2), (288, 8, 32, 4, 2), (384, 8, 1, 1, 1), (100, 7, 4, 4, 2), (512, 10, 16, 5, 2),
    (640, 3, 2, 1, 1), (1000, 8, 1, 1, 1), (1024, 32, 32, 7, 2), (12, 2, 4, 2, 1)]


@pytest.mark.parametrize("score,biased,renormalize", list(itertools.product(["softmax", "sigmoid"], [False, True], [True, False])))
@pytest.mark.parametrize("E,k,G,tg,gt", SHAPES)
def test_route(E, k, G, tg, gt, score, biased, renormalize):
    rng = np.random.default_rng([E, k, G, biased])
    T = 131
    bias = rng.standard_normal(E) * 0.1 if biased else None
    for dtype in DT:
        _check(rng.standard_normal((T, E)) * 1.5, k, dtype, bias, score=score, renormalize=renormalize, groups=G, topk_groups=tg,
               group_top=gt, scale=2.5)


@pytest.mark.parametrize("T", [1, 3, 4, 5, 8192])
def test_token_counts(T):
    rng = np.random.default_rng(T)
    _check(rng.standard_normal((T, 64)), 4, bias=rng.standard_normal(64) * 0.1, score="sigmoid")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [(1, 1, 1), (4, 2, 2)])
def test_keys_closer_than_fp32_tells_apart(score, groups):
    """Scores and biases whose sums differ by 1e-9 to 1e-6 from one expert to the next, in shuffled order:
    the order is that of the sums in 64 bits."""
    G, tg, gt = groups
    rng = np.random.default_rng(5)
    T, E = 64, 64
    for gap in (1e-9, 1e-8, 1e-7, 1e-6):
        logits = rng.standard_normal((T, E)).astype(np.float32)
        # one bias serves all tokens, so each token's logits are set from the key it is to have
        bias = (rng.standard_normal(E) * 0.05).astype(np.float32)
        for t in range(T):
            p = 0.3 + rng.permutation(E) * gap - bias.astype(np.float64)      # scores wanted
            logits[t] = np.log(p / (1 - p)) if score == "sigmoid" else np.log(p)
        _check(logits, 8, bias=bias, score=score, groups=G, topk_groups=tg, group_top=gt)


def test_ties_go_to_the_lower_expert_and_group():
    from mosaicist_b200 import ops

    x = torch.zeros(5, 64, device="cuda")
    x[1, 40] = x[1, 7] = 3.0
    for kw in (dict(), dict(score="sigmoid"), dict(bias=torch.zeros(64, device="cuda")),
               dict(score="sigmoid", bias=torch.full((64,), 0.25, device="cuda"))):
        ids, w = ops.moe_route(x, 3, **kw)
        assert ids[0].tolist() == [0, 1, 2] and ids[1].tolist() == [7, 40, 0]
        assert torch.equal(w[0], torch.full((3,), 1 / 3, device="cuda"))
        ids, _ = ops.moe_route(x, 3, groups=8, topk_groups=2, group_top=2, **kw)
        assert ids[0].tolist() == [0, 1, 2] and ids[1].tolist() == [7, 40, 0]
    # saturated scores are equal although the logits are not: with a bias the sums tie, without one the
    # logits decide
    x = torch.full((1, 8), 40.0, device="cuda")
    x[0, 5] = 60.0
    assert ops.moe_route(x, 1, score="sigmoid")[0].item() == 5
    assert ops.moe_route(x, 1, score="sigmoid", bias=torch.zeros(8, device="cuda"))[0].item() == 0


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_barred_experts(score, biased, renormalize):
    """Logits of -inf and NaN, biases of -inf: barred; rows that leave fewer than topk, one, or nothing."""
    rng = np.random.default_rng(11)
    T, E = 40, 96
    x = rng.standard_normal((T, E))
    bias = rng.standard_normal(E) * 0.1 if biased else None
    if biased:
        bias[17] = -np.inf
        bias[18] = np.nan
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 1:] = -np.inf
    x[3, :90] = -np.inf
    x[4, 5:] = np.nan
    x[5] = np.finfo(np.float32).min
    x[6, ::2] = np.finfo(np.float32).min
    x[7] = 1e4
    x[8, 3] = 1e30
    x[9, rng.permutation(E)[:50]] = -np.inf
    for kw in (dict(), dict(groups=8, topk_groups=3, group_top=1), dict(groups=8, topk_groups=3, group_top=2)):
        seen, ids, w = _check(x, 7, "f32", bias, score=score, renormalize=renormalize, **kw)
        got = ids.cpu().numpy()
        assert all(len(set(r)) == 7 for r in got.tolist()) and got.min() >= 0 and got.max() < E
        assert torch.isfinite(w).all() and (w[0] == 0).all() and (w[1] == 0).all()


def test_infinite_logits():
    x = np.zeros((3, 40))
    x[0, 9] = np.inf
    x[1, [4, 30]] = np.inf
    x[2] = np.inf
    for score in ("softmax", "sigmoid"):
        for bias in (None, np.zeros(40)):
            _check(x, 3, bias=bias, score=score, renormalize=False)


def test_infinite_bias_comes_first():
    x = np.random.default_rng(0).standard_normal((16, 64))
    bias = np.zeros(64)
    bias[[50, 60]] = np.inf
    _, ids, _ = _run(x, 4, bias=bias, score="sigmoid")
    assert (ids[:, :2].cpu().numpy() == [50, 60]).all()


@pytest.mark.parametrize("score,renormalize", list(itertools.product(["softmax", "sigmoid"], [True, False])))
@pytest.mark.parametrize("E,k", [(1, 1), (33, 4), (61, 4), (160, 6), (256, 8), (1024, 32)])
def test_backward(E, k, score, renormalize):
    from mosaicist_b200 import ops

    rng = np.random.default_rng([E, k])
    T, scale = 77, 2.5
    for dtype in DT:
        x = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)).to(DT[dtype]).cuda()
        ids, w = ops.moe_route(x, k, score=score, renormalize=renormalize, scale=scale)
        g = torch.from_numpy(rng.standard_normal((T, k)).astype(np.float32)).cuda()
        got = ops.moe_route_backward(g, x, ids, w, score=score, renormalize=renormalize, scale=scale)
        assert got.dtype == x.dtype and got.shape == x.shape
        xs, i, ws, gs = x.float().cpu().numpy(), ids.cpu().numpy(), w.cpu().numpy(), g.cpu().numpy()
        want = R.route_backward(gs, xs, i, ws, score, renormalize, scale)
        # sum g w and what it meets: the terms' magnitudes times (additions, exponential, quotient)
        terms = np.abs(gs * ws).sum(1, keepdims=True)
        part = np.take_along_axis(np.zeros_like(want), i, axis=1) + np.abs(ws) * (np.abs(gs) + terms / scale)
        bound = np.zeros_like(want)
        np.put_along_axis(bound, i, part, axis=1)
        if score == "softmax" and not renormalize:
            bound += R.scores(xs, score) * terms
        out = got.float().cpu().numpy()
        assert (np.abs(out - want) <= EPS[dtype] * np.abs(want) + 80 * 2.0 ** -24 * bound + (2.0 ** -25 if dtype == "f16" else 0)).all()


@pytest.mark.parametrize("score,renormalize", list(itertools.product(["softmax", "sigmoid"], [True, False])))
def test_backward_against_differences(score, renormalize):
    """The kernel's gradient against central differences of the weights in 64 bits, the choice held."""
    from mosaicist_b200 import ops

    rng = np.random.default_rng(3)
    T, E, k, scale, h = 5, 24, 4, 1.5, 1e-5
    x = rng.standard_normal((T, E)).astype(np.float32)
    g = rng.standard_normal((T, k)).astype(np.float32)
    xt = torch.from_numpy(x).cuda()
    ids, w = ops.moe_route(xt, k, score=score, renormalize=renormalize, scale=scale)
    got = ops.moe_route_backward(torch.from_numpy(g).cuda(), xt, ids, w, score=score, renormalize=renormalize, scale=scale).cpu().numpy()
    i, x64 = ids.cpu().numpy(), x.astype(np.float64)
    for e in range(E):
        d = np.zeros((T, E))
        d[:, e] = h
        diff = (R.weights_of(x64 + d, i, score, renormalize, scale) - R.weights_of(x64 - d, i, score, renormalize, scale)) / (2 * h)
        # h^2 / 6 of the third derivative (below 1 here) and fp32's share of the result
        assert np.abs(got[:, e] - (g * diff).sum(1)).max() <= 4 * scale * np.abs(g).max() * (h * h + 80 * 2.0 ** -24)


def test_backward_of_barred_and_repeated_ids():
    from mosaicist_b200 import ops

    x = torch.randn(6, 40, device="cuda")
    x[0] = -torch.inf
    x[1, 2:] = -torch.inf
    for score, renorm in itertools.product(("softmax", "sigmoid"), (True, False)):
        ids, w = ops.moe_route(x, 4, score=score, renormalize=renorm)
        g = torch.randn(6, 4, device="cuda")
        g[0] = torch.inf                   # weights of 0 do not move
        got = ops.moe_route_backward(g, x, ids, w, score=score, renormalize=renorm)
        want = R.route_backward(g.cpu().numpy(), x.cpu().numpy(), ids.cpu().numpy(), w.cpu().numpy(), score, renorm, 1.0)
        assert torch.isfinite(got).all() and (got[0] == 0).all()
        assert np.abs(got.cpu().numpy() - want).max() <= 80 * 2.0 ** -24 * 16
    # an id twice collects both shares; ids that are no expert are skipped
    ids = torch.tensor([[3, 3, 7, 0]] * 6, dtype=torch.int32, device="cuda")
    w = torch.full((6, 4), 0.25, device="cuda")
    x = torch.randn(6, 40, device="cuda")
    got = ops.moe_route_backward(g.nan_to_num(1, 1, 1), x, ids, w, score="sigmoid", renormalize=False)
    want = R.route_backward(g.nan_to_num(1, 1, 1).cpu().numpy(), x.cpu().numpy(), ids.cpu().numpy(), w.cpu().numpy(), "sigmoid", False, 1.0)
    assert np.abs(got.cpu().numpy() - want).max() <= 80 * 2.0 ** -24 * 16
    ids[:, 3] = -1
    ids[:, 2] = 40
    got = ops.moe_route_backward(g.nan_to_num(1, 1, 1), x, ids, w, score="sigmoid", renormalize=False)
    assert (got[:, :3] == 0).all() and (got[:, 4:] == 0).all() and (got[:, 3] != 0).all()


def test_out_buffers_streams_and_graphs():
    from mosaicist_b200 import ops

    x, b = torch.randn(300, 128, device="cuda"), torch.randn(128, device="cuda") * 0.1
    kw = dict(score="sigmoid", bias=b, groups=4, topk_groups=2, group_top=2)
    want = ops.moe_route(x, 6, **kw)
    out = (torch.empty(300, 6, dtype=torch.int32, device="cuda"), torch.empty(300, 6, device="cuda"))
    got = ops.moe_route(x, 6, out=out, **kw)
    assert got[0].data_ptr() == out[0].data_ptr() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = ops.moe_route(x, 6, **kw)
        grad = ops.moe_route_backward(again[1], x, *again, score="sigmoid")
    s.synchronize()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = ops.moe_route(x, 6, **kw)
        held_grad = ops.moe_route_backward(held[1], x, *held, score="sigmoid")
    x.copy_(x.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], want[0].flip(0)) and torch.equal(held[1], want[1].flip(0))
    assert torch.equal(held_grad, grad.flip(0))
    assert ops.moe_route(x[:0], 6, **kw)[0].shape == (0, 6)
    assert ops.moe_route_backward(want[1][:0], x[:0], want[0][:0], want[1][:0]).shape == (0, 128)


def test_torch_operators():
    import mosaicist_b200.torch_ops as T
    from mosaicist_b200 import ops

    x, b = torch.randn(33, 64, device="cuda"), torch.randn(64, device="cuda") * 0.1
    got = T.moe_route(x, 4, "sigmoid", b, 8, 3, 2, True, 2.0)
    want = ops.moe_route(x, 4, "sigmoid", b, 8, 3, 2, True, 2.0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    d = T.moe_route_backward(got[1], x, *got, "sigmoid", True, 2.0)
    assert torch.equal(d, ops.moe_route_backward(got[1], x, *got, score="sigmoid", scale=2.0))


def test_the_layers_own_routing_is_the_plain_case():
    """msc_moe_route_topk and moe_route with its defaults make the same choices."""
    from mosaicist_b200 import _lib, ops

    x = torch.randn(500, 256, device="cuda")
    ids, w = torch.empty(500, 8, dtype=torch.int32, device="cuda"), torch.empty(500, 8, device="cuda")
    _lib.check(_lib.load().msc_moe_route_topk(x.data_ptr(), ids.data_ptr(), w.data_ptr(), 500, 256, 8,
                                              torch.cuda.current_stream().cuda_stream))
    got = ops.moe_route(x, 8)
    assert torch.equal(got[0], ids)
    assert (got[1] - w).abs().max() <= 2e-6


# From 1024 tokens on eight lanes share a token of up to 256 experts (1, 2, 4 or 8 groups, topk up to 8).
MANY = [  # experts, topk, groups, topk_groups, group_top
    (1, 1, 1, 1, 1), (2, 2, 1, 1, 1), (7, 3, 1, 1, 1), (8, 8, 8, 8, 1), (8, 4, 8, 5, 1), (16, 3, 2, 1, 2), (31, 5, 1, 1, 1), (61, 4, 1, 1, 1),
    (64, 8, 4, 2, 2), (100, 7, 4, 3, 2), (128, 8, 1, 1, 1), (130, 6, 2, 1, 2), (160, 6, 8, 3, 1), (160, 8, 8, 3, 2), (200, 1, 8, 1, 2), (250, 8, 2, 1, 1),
    (255, 7, 1, 1, 1), (256, 8, 8, 4, 2), (256, 8, 8, 1, 2), (256, 8, 4, 2, 1), (256, 1, 1, 1, 1)]


@pytest.mark.parametrize("score,biased,renormalize", list(itertools.product(["softmax", "sigmoid"], [False, True], [True, False])))
@pytest.mark.parametrize("E,k,G,tg,gt", MANY)
def test_many_tokens(E, k, G, tg, gt, score, biased, renormalize):
    rng = np.random.default_rng([E, k, G, biased, 1])
    bias = rng.standard_normal(E) * 0.1 if biased else None
    for dtype, T in (("f32", 1027), ("bf16", 1025), ("f16", 1030)):
        _check(rng.standard_normal((T, E)) * 1.5, k, dtype, bias, score=score, renormalize=renormalize, groups=G, topk_groups=tg,
               group_top=gt, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [(1, 1, 1), (4, 2, 2), (8, 3, 1)])
def test_many_tokens_with_keys_closer_than_fp32_tells_apart(score, groups):
    G, tg, gt = groups
    rng = np.random.default_rng(6)
    T, E = 1024, 64
    for gap in (1e-9, 1e-7, 1e-6, 4e-6):
        bias = (rng.standard_normal(E) * 0.05).astype(np.float32)
        p = 0.3 + rng.permuted(np.tile(np.arange(E), (T, 1)), axis=1) * gap - bias.astype(np.float64)
        logits = (np.log(p / (1 - p)) if score == "sigmoid" else np.log(p)).astype(np.float32)
        _check(logits, 8, bias=bias, score=score, groups=G, topk_groups=tg, group_top=gt)
        _check(logits, 7, score=score, groups=G, topk_groups=tg, group_top=gt)       # the logits themselves


def _undecided(x, score, bias, groups, topk_groups, group_top):
    """Tokens whose choice hangs on the last bits of 64-bit arithmetic: two groups (one in, one out) or two
    experts of which different logits and biases make sums that are equal to 2^-46.  (Equal logits with equal
    biases are a tie in any arithmetic, and decided.)  A score is off by at most 2 ulp of its exponential, the
    sum of up to 96 terms and a quotient, and its sums with biases of magnitude < 2 by 2^-52 each: less than
    110 x 2^-53 < 2^-46."""
    near, out = 2.0 ** -46, np.zeros(len(x), bool)
    b = np.zeros(x.shape[1]) if bias is None else bias
    key = R.scores(x, score) + b
    E = x.shape[1]
    for t in range(len(x)):
        allowed = np.ones(E, bool)
        if topk_groups < groups:
            order = np.argsort(-key[t].reshape(groups, -1), axis=1, kind="stable")[:, :group_top] + np.arange(groups)[:, None] * (E // groups)
            strength = key[t][order].sum(axis=1)
            what = [sorted(zip(x[t, o], b[o])) for o in order]
            kept = set(np.argsort(-strength, kind="stable")[:topk_groups].tolist())
            for g in kept:
                for h in set(range(groups)) - kept:
                    out[t] |= abs(strength[g] - strength[h]) <= near and what[g] != what[h]
            allowed = np.isin(np.arange(E) // (E // groups), list(kept))
        at = np.flatnonzero(allowed)
        at = at[np.argsort(-key[t, at], kind="stable")]
        gap = key[t, at][:-1] - key[t, at][1:]
        differ = (x[t, at][:-1] != x[t, at][1:]) | (b[at][:-1] != b[at][1:])
        out[t] |= bool(((gap <= near) & differ).any())
    return out


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 3, 1), (8, 3, 2), (2, 1, 2)])
def test_many_tokens_with_ties_and_zeros(score, groups):
    G, tg, gt = groups
    rng = np.random.default_rng(7)
    x = np.round(rng.standard_normal((1500, 96)) * 2) / 2     # few different values: ties within and across lanes
    x[0:40] = 0.0
    x[40:80, ::3] = -0.0                                      # equal to 0
    x[80:90] = 88.0
    x[90:100] = -200.0
    for dtype in DT:
        for bias in (None, np.zeros(96), np.round(rng.standard_normal(96)) / 4):
            if bias is None and (gt == 1 or G == 1):      # the logits decide
                _check(x, 8, dtype, bias, score=score, groups=G, topk_groups=tg, group_top=gt)
                continue
            seen, ids, w = _run(x, 8, dtype, bias, score=score, groups=G, topk_groups=tg, group_top=gt)
            want, want_w = R.route(seen, 8, score, bias, groups=G, topk_groups=tg, group_top=gt)
            sure = ~_undecided(seen, score, bias, G, tg, gt)
            assert sure.sum() > 1350
            assert np.array_equal(ids.cpu().numpy()[sure], want[sure])
            assert (np.abs(w.cpu().numpy() - want_w) <= W_TOL * want_w + 2.0 ** -126)[sure].all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [(1, 1, 1), (8, 3, 1), (8, 4, 2)])
@pytest.mark.parametrize("kind", ["far", "masked", "lowest", "both ends", "few left", "none left", "inf", "offset"])
def test_many_tokens_with_wide_biases(kind, groups, score):
    """Biases that span more than the scores do, masks made of biases, biases that bar."""
    G, tg, gt = groups
    rng = np.random.default_rng(8)
    E = 96
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32)
    if kind == "far":
        bias *= 100
    elif kind == "masked":
        bias[rng.permutation(E)[:80]] = -1e9
    elif kind == "lowest":
        bias[rng.permutation(E)[:90]] = np.finfo(np.float32).min
    elif kind == "both ends":
        bias[::2] = np.finfo(np.float32).min
        bias[1::24] = np.finfo(np.float32).max
    elif kind == "few left":
        bias[5:] = -np.inf
    elif kind == "none left":
        bias[:] = np.where(np.arange(E) % 2, -np.inf, np.nan)
    elif kind == "inf":
        bias[[3, 50, 51]] = np.inf
    elif kind == "offset":
        bias += 1000.0
    _check(rng.standard_normal((1024, E)) * 1.5, 8, "f32", bias, score=score, groups=G, topk_groups=tg, group_top=gt)


@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("score,biased", list(itertools.product(["softmax", "sigmoid"], [False, True])))
def test_many_tokens_with_barred_and_infinite_logits(score, biased, renormalize):
    rng = np.random.default_rng(9)
    T, E = 1100, 96
    x = rng.standard_normal((T, E))
    x[:900:9] = -np.inf
    x[1:900:9] = np.nan
    x[2:900:9, 1:] = -np.inf
    x[3:900:9, :90] = -np.inf
    x[4:900:9, 5:] = np.nan
    x[5:900:9] = np.finfo(np.float32).min
    x[6:900:9, ::2] = np.finfo(np.float32).min
    x[7:900:9] = 1e4
    x[8:900:9, 3] = 1e30
    x[1000:1020, [7, 60]] = np.inf
    bias = rng.standard_normal(E) * 0.1 if biased else None
    for kw in (dict(), dict(groups=8, topk_groups=3, group_top=1), dict(groups=8, topk_groups=3, group_top=2)):
        _check(x, 7, "f32", bias, score=score, renormalize=renormalize, **kw)


@pytest.mark.parametrize("T", [20, 1040])
def test_sigmoids_that_vanish_in_32_bits(T):
    """Their ratios do not; those that vanish in 64 bits too leave nothing to divide."""
    rng = np.random.default_rng(10)
    x = np.round(rng.standard_normal((T, 64)) * 2)
    x -= np.array([60, 64, 65, 90, 104, 200, 650, 700])[np.arange(T) % 8, None]
    _check(x, 6, score="sigmoid")
    _check(x, 6, score="sigmoid", groups=8, topk_groups=3, group_top=1)
    _check(np.full((T, 64), -710.0), 6, score="sigmoid")


def test_a_token_routes_alike_alone_and_among_many():
    from mosaicist_b200 import ops

    x = torch.randn(2000, 256, device="cuda")
    bias = torch.randn(256, device="cuda") * 0.1
    kw = dict(bias=bias, score="sigmoid", groups=8, topk_groups=4, group_top=2)
    ids, w = ops.moe_route(x, 8, **kw)
    for t in (0, 3, 1024, 1999):
        one, ow = ops.moe_route(x[t:t + 1], 8, **kw)
        assert torch.equal(one[0], ids[t]) and torch.allclose(ow[0], w[t], rtol=8 * 2.0 ** -24, atol=0)   # (the sum's order)


def test_backward_with_a_tiny_scale():
    """The quotient by the scale is one even where its reciprocal is not a number."""
    from mosaicist_b200 import ops

    scale = 1e-39
    x = torch.randn(3, 16, device="cuda")
    ids, w = ops.moe_route(x, 4, scale=scale)
    g = torch.randn(3, 4, device="cuda")
    dx = ops.moe_route_backward(g, x, ids, w, scale=scale)
    assert torch.isfinite(dx).all() and float(dx.abs().max()) <= 8 * scale


@pytest.mark.parametrize("masks", [0, 10])
@pytest.mark.parametrize("groups", [(1, 1, 1), (2, 2, 1), (4, 3, 1), (4, 3, 2)])
@pytest.mark.parametrize("E", [16, 32])
def test_many_tokens_with_close_keys_beside_barred_biases(E, groups, masks):
    """Sigmoids that fall together at the lower end of the keys' window, so that every expert comes into question and
    is ranked in 64 bits, but for those that a NaN or -inf bias bars."""
    G, tg, gt = groups
    rng = np.random.default_rng([E, G, gt, masks])
    T = 1025
    bias = np.zeros(E, np.float32)
    at = rng.permutation(E)
    bias[at[2:2 + masks]] = -1e9
    bias[at[0]], bias[at[1]] = np.nan, -np.inf
    for far in (-30.0, 0.0):
        x = rng.standard_normal((T, E)) + far
        _, ids, w = _check(x, 8 if G == 1 else 6, "f32", bias, score="sigmoid", groups=G, topk_groups=tg, group_top=gt)
        got = ids.cpu().numpy()
        assert not np.isin(got, at[:2]).any()
        assert all(len(set(r)) == len(r) for r in got.tolist())


@pytest.mark.parametrize("T", [20, 1040])
def test_sigmoids_of_which_some_vanish_in_32_bits(T):
    """The best choice is an ordinary number, others are sub-normal or 0 in fp32; their share of the sum is not."""
    rng = np.random.default_rng(11)
    x = np.full((T, 64), -400.0)
    best = np.array([-10, -16, -17, -20, -40, -60, -63, -64])[np.arange(T) % 8]
    x[:, 3] = best
    for e, lo, hi in ((7, -96, -87), (20, -103, -96), (21, -110, -103), (40, -130, -110), (61, -90, -70)):
        x[:, e] = rng.integers(lo, hi, T)
    _check(x, 6, score="sigmoid")
    _check(x, 6, score="sigmoid", scale=2.5, bias=np.zeros(64))


def test_an_empty_batch_with_a_wrong_configuration():
    from mosaicist_b200 import _lib, ops

    x, ids, w = torch.empty(0, 64, device="cuda"), torch.empty(0, 4, dtype=torch.int32, device="cuda"), torch.empty(0, 4, device="cuda")
    assert ops.moe_route(x, 4)[0].shape == (0, 4) and ops.moe_route_backward(w, x, ids, w).shape == (0, 64)
    for kw in (dict(groups=3), dict(groups=8, topk_groups=9), dict(group_top=3), dict(scale=-1.0)):
        with pytest.raises(_lib.MscError):
            ops.moe_route(x, 4, **kw)
    with pytest.raises(_lib.MscError):
        ops.moe_route_backward(w, x, ids, w, scale=0.0)


@pytest.mark.parametrize("score,renormalize,dtype", [("softmax", True, "f32"), ("softmax", False, "bf16"), ("sigmoid", True, "f16"), ("sigmoid", False, "f32")])
def test_weights_carry_the_gradient_on(score, renormalize, dtype):
    """ops.moe_route and the torch operator inside a graph of gradients: moe_route_backward's result, also of an expanded
    gradient; captured and replayed on new data."""
    import mosaicist_b200.torch_ops as O
    from mosaicist_b200 import ops

    kw = dict(score=score, groups=4, topk_groups=2, group_top=2, renormalize=renormalize, scale=2.5)
    bias = torch.randn(64, device="cuda") * 0.1
    x = torch.randn(300, 64, device="cuda").to(DT[dtype]).requires_grad_()
    g = torch.randn(300, 6, device="cuda")
    want_ids, want_w = ops.moe_route(x.detach(), 6, bias=bias, **kw)
    back = lambda grad, v, ids, w: ops.moe_route_backward(grad, v, ids, w, score, renormalize, 2.5)
    for ids, w in (ops.moe_route(x, 6, bias=bias, **kw), O.moe_route(x, 6, score, bias, 4, 2, 2, renormalize, 2.5)):
        assert torch.equal(ids, want_ids) and torch.equal(w, want_w) and w.requires_grad and not ids.requires_grad
        assert torch.equal(torch.autograd.grad(w, x, g, retain_graph=True)[0], back(g, x.detach(), ids, want_w))
        assert torch.equal(torch.autograd.grad(w.sum(), x)[0], back(torch.ones_like(g), x.detach(), ids, want_w))
    with torch.no_grad():
        assert not ops.moe_route(x, 6, bias=bias, **kw)[1].requires_grad
    del w, ids
    leaf = x.detach().clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.moe_route(leaf, 6, bias=bias, **kw)[1], leaf, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, w = ops.moe_route(leaf, 6, bias=bias, **kw)
        held = torch.autograd.grad(w, leaf, g)[0]
        w = w.detach()
    with torch.no_grad():
        leaf.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ids, want_ids.flip(0)) and torch.equal(held, back(g, x.detach().flip(0).contiguous(), ids, w))
