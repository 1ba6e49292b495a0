"""The routed layer over FP8 weights with fp32 scales per block of 128: dispatch bit for bit, the layer against the
oracle, and the run of its operators together."""

import ml_dtypes
import numpy as np
import pytest
import torch

from oracle import fp8_block as F, moe as M, route as R

pytestmark = pytest.mark.gpu


def T(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    from mosaicist_b200 import _lib

    assert _lib.status_word() == 0


def _weights(E, h, n, seed):
    rng = np.random.default_rng([seed, 0])
    w1 = [F.quantize_weight((rng.standard_normal((2 * n, h)) * 0.05).astype(np.float32)) for _ in range(E)]
    w2 = [F.quantize_weight((rng.standard_normal((h, n)) * 0.05).astype(np.float32)) for _ in range(E)]
    return tuple(np.stack(v) for v in zip(*w1)) + tuple(np.stack(v) for v in zip(*w2))


def _bf16(x):
    return x.astype(ml_dtypes.bfloat16).astype(np.float64)


def _layer(tokens, ids, weights, w, first=0):
    """(T, h) float64: every step as the layer defines it, products and activation in 64 bits."""
    w1_q, w1_sf, w2_q, w2_sf = w
    out = np.zeros(tokens.shape)
    for e in range(len(w1_q)):
        t, k = np.nonzero(ids == e + first)
        if not len(t):
            continue
        gateup = _bf16(F.product(*F.quantize_rows(tokens[t]), w1_q[e], w1_sf[e])[0])
        y = F.product(*F.quantize_rows(F.silu_mul(gateup).astype(np.float32)), w2_q[e], w2_sf[e])[0]
        np.add.at(out, t, _bf16(y * weights[t, k][:, None]))
    return out


def _close(got, want):
    """Of the largest value: 3 % at most, 0.3 % in the mean square.  A product that is rounded the other way to bf16
    (2^-8) can move an activation by a whole e4m3 step (2^-3) in the second quantisation; that is one of n
    terms of a result, each a fraction of it."""
    scale = np.abs(want).max()
    off = np.abs(got - want) / scale
    assert off.max() < 3e-2 and np.sqrt((off ** 2).mean()) < 3e-3, (off.max(), np.sqrt((off ** 2).mean()))
    assert np.count_nonzero(want) > 0.5 * want.size


@pytest.mark.parametrize("tokens,h,E,k,first,local", [(200, 256, 32, 4, 0, 32), (90, 400, 16, 3, 4, 8), (1, 7168, 8, 2, 0, 8), (700, 1040, 8, 2, 0, 8)])
def test_dispatch_bit_exact(tokens, h, E, k, first, local):
    from mosaicist_b200 import _lib

    rng = np.random.default_rng([tokens, h])
    ids, w = M.route_topk(rng.standard_normal((tokens, E)).astype(np.float32), k)
    x = rng.standard_normal((tokens, h)).astype(np.float32).astype(ml_dtypes.bfloat16)
    rank, rows, offs, total = M.plan(ids, first, local)
    cap = (tokens * k + 127 * local + 127) // 128 * 128
    q = torch.full((cap, h), 0x55, dtype=torch.uint8, device="cuda")
    sf = torch.full((-(-h // 128), cap), -7.0, device="cuda")
    rw, rt = torch.full((cap,), -1.0, device="cuda"), torch.full((cap,), -1, dtype=torch.int32, device="cuda")
    # (an ABI call keeps its tensors alive itself)
    held = [T(x.view(np.int16)), T(ids), T(w), T(rank), T(offs)]
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.load().msc_moe_permute_quantize_fp8_block(*(t.data_ptr() for t in held), tokens, h, k, first, local, q.data_ptr(),
                                                              sf.data_ptr(), rw.data_ptr(), rt.data_ptr(), cap, st))
    want_q, want_sf = F.quantize_rows(x.astype(np.float32))
    q, sf, rw, rt = (t.cpu().numpy() for t in (q, sf, rw, rt))
    live = np.zeros(cap, bool)
    for t in range(tokens):
        for j in range(k):
            e = ids[t, j] - first
            if 0 <= e < local:
                r = offs[e] + rank[t, j]
                live[r] = True
                assert np.array_equal(q[r], want_q[t]) and np.array_equal(sf[:, r], want_sf[:, t])
                assert rw[r] == w[t, j] and rt[r] == t
    assert live.sum() == rows.sum() and (q[~live] == 0x55).all() and (sf[:, ~live] == -7).all() and (rt[~live] == -1).all()


ROUTES = [dict(), dict(score="sigmoid", groups=2, topk_groups=1, group_top=2, scale=2.5), dict(renormalize=False, scale=16.0)]


@pytest.mark.parametrize("route", range(len(ROUTES)))
@pytest.mark.parametrize("tokens,h,n,E,k", [(1, 256, 128, 8, 2), (33, 272, 144, 16, 4), (300, 512, 256, 8, 2), (700, 256, 384, 4, 2)])
def test_layer(tokens, h, n, E, k, route):
    from mosaicist_b200.moe import MegaMoEFp8Block, RouteConfig

    cfg = ROUTES[route]
    rng = np.random.default_rng([tokens, h, n])
    w = _weights(E, h, n, tokens)
    x = rng.standard_normal((tokens, h)).astype(np.float32).astype(ml_dtypes.bfloat16)
    logits = rng.standard_normal((tokens, E)).astype(np.float32)
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32) if route == 1 else None
    ids, weights = R.route(logits, k, bias=bias, **cfg)
    weights = weights.astype(np.float32).astype(np.float64)
    want = _layer(x.astype(np.float32), ids, weights, w)
    dev = [T(v) for v in w]
    layer = MegaMoEFp8Block(*dev, topk=k, max_tokens=tokens + 5, route=RouteConfig(**cfg), route_bias=None if bias is None else T(bias))
    tx, tl = T(x.view(np.int16)).view(torch.bfloat16), T(logits)
    got = layer.forward(tx, tl)
    assert np.array_equal(layer.ids[:tokens].cpu().numpy(), ids)
    _close(got.double().cpu().numpy(), want)
    # a smaller call on the same workspaces, and the first one again from the routing it left
    if tokens > 1:
        _close(layer.forward(tx[:tokens // 2], tl[:tokens // 2]).double().cpu().numpy(), want[:tokens // 2])
        layer.route(tl)
        assert torch.equal(layer.forward(tx), got)
    assert layer.forward(tx[:0], tl[:0]).shape == (0, h)


def test_shares_of_the_experts_add_up():
    from mosaicist_b200.moe import MegaMoEFp8Block

    rng = np.random.default_rng(4)
    E, h, n, k, tokens = 8, 256, 128, 3, 50
    w = _weights(E, h, n, 1)
    x = rng.standard_normal((tokens, h)).astype(np.float32).astype(ml_dtypes.bfloat16)
    logits = rng.standard_normal((tokens, E)).astype(np.float32)
    ids, weights = R.route(logits, k)
    got = np.zeros((tokens, h))
    for first in (0, 4):
        part = tuple(v[first:first + 4] for v in w)
        layer = MegaMoEFp8Block(*(T(v) for v in part), topk=k, max_tokens=tokens, expert_first=first)
        mine = layer.forward(T(x.view(np.int16)).view(torch.bfloat16), T(logits)).double().cpu().numpy()
        want = _layer(x.astype(np.float32), ids, weights.astype(np.float32).astype(np.float64), part, first)
        scale = np.abs(want).max()
        assert np.abs(mine - want).max() < 3e-2 * scale
        got += mine
    _close(got, _layer(x.astype(np.float32), ids, weights.astype(np.float32).astype(np.float64), w))


def test_layer_in_a_graph():
    from mosaicist_b200.moe import MegaMoEFp8Block, RouteConfig

    E, h, n, k, tokens = 8, 512, 256, 2, 64
    layer = MegaMoEFp8Block(*(T(v) for v in _weights(E, h, n, 2)), topk=k, max_tokens=tokens, route=RouteConfig(score="sigmoid"),
                            route_bias=torch.randn(E, device="cuda") * 0.1)
    x, logits = torch.randn(tokens, h, device="cuda").bfloat16(), torch.randn(tokens, E, device="cuda")
    layer.forward(x, logits)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer.forward(x, logits)
    for _ in range(3):
        x.copy_(torch.randn(tokens, h, device="cuda"))
        logits.copy_(torch.randn(tokens, E, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        held = out.clone()
        assert torch.equal(held, layer.forward(x, logits))


def test_the_nvfp4_layer_takes_a_route_config():
    """MegaMoE with a RouteConfig: the experts and weights of ops.moe_route, the layer as without one."""
    from mosaicist_b200 import ops
    from mosaicist_b200.moe import MegaMoE, RouteConfig

    E, h, n, k, tokens = 32, 256, 256, 4, 70
    g = torch.Generator(device="cuda").manual_seed(0)
    w1, w2 = (0.05 * torch.randn(s, device="cuda", generator=g) for s in ((E, 2 * n, h), (E, h, n)))
    ones = torch.ones(E, device="cuda")
    gs1, gs2 = ops.global_scale_for(w1), ops.global_scale_for(w2)
    args = (*ops.quantize_nvfp4(w1, gs1), gs1, ones, *ops.quantize_nvfp4(w2, gs2), gs2, ones, 300 * ones, 300 * ones)
    x, logits = torch.randn(tokens, h, device="cuda", generator=g).bfloat16(), torch.randn(tokens, E, device="cuda", generator=g)
    bias = 0.1 * torch.randn(E, device="cuda", generator=g)
    cfg = RouteConfig(score="sigmoid", groups=8, topk_groups=4, group_top=2, scale=2.0)
    plain = MegaMoE(*args, topk=k, max_tokens=tokens)
    routed = MegaMoE(*args, topk=k, max_tokens=tokens, route=cfg, route_bias=bias)
    got = routed.forward(x, logits)
    ids, w = ops.moe_route(logits, k, "sigmoid", bias, 8, 4, 2, True, 2.0)
    assert torch.equal(routed.ids, ids) and torch.equal(routed.weights, w)
    plain.ids.copy_(ids)
    plain.weights.copy_(w)
    assert torch.equal(plain.forward(x), got)
    assert not torch.equal(plain.forward(x, logits), got)
    with pytest.raises(ValueError):
        routed.forward(x, logits[:-1])


def test_one_expert_parallel_rank_equals_the_layer():
    """ExpertParallelMoE of one rank over an FP8 layer with a router of its own: the layer's result, bit for bit."""
    import torch.distributed as dist

    from mosaicist_b200.moe import MegaMoEFp8Block, RouteConfig
    from mosaicist_b200.parallel import ExpertParallelMoE

    E, h, n, k, tokens = 8, 256, 128, 3, 50
    w = [T(v) for v in _weights(E, h, n, 5)]
    cfg = RouteConfig(score="sigmoid", groups=2, topk_groups=1, group_top=2, scale=2.5)
    bias = torch.randn(E, device="cuda") * 0.2
    x, logits = torch.randn(tokens, h, device="cuda").bfloat16(), torch.randn(tokens, E, device="cuda").bfloat16()
    want = MegaMoEFp8Block(*w, topk=k, max_tokens=tokens, route=cfg, route_bias=bias).forward(x, logits)
    dist.init_process_group("nccl", store=dist.HashStore(), rank=0, world_size=1, device_id=torch.device("cuda", 0))
    try:
        share = MegaMoEFp8Block(*w, topk=1, max_tokens=tokens * k, route=cfg, route_bias=bias)
        assert torch.equal(ExpertParallelMoE(share, E, k).forward(x, logits), want)
    finally:
        dist.destroy_process_group()


def _in_rows_cap(ids, first, local, cap):
    """The pairs that fit, the others' ids -1 (later rows of an expert are later tokens', so the ranks stay)."""
    rank, rows, offs, _ = M.plan(ids, first, local)
    e = ids - first
    here = (e >= 0) & (e < local)
    fits = here & (offs[np.where(here, e, 0)] + np.where(here, rank, 0) < cap)
    assert (here & ~fits).any() and fits.any()
    return np.where(fits, ids, -1).astype(np.int32)


def _guarded(rows, cols, dtype, fill):
    """A buffer of `rows` rows with 64 rows behind it that nobody may read or write."""
    whole = torch.empty((rows + 64, cols) if cols else (rows + 64,), dtype=dtype, device="cuda")
    whole.fill_(fill)
    return whole, whole[:rows]


def test_a_small_rows_cap_leaves_pairs_out():
    """More rows than rows_cap: nothing is read or written behind the buffers, the pairs that do not fit are missing from
    the sum and the status word says so."""
    from mosaicist_b200 import _lib
    from mosaicist_b200.moe import MegaMoEFp8Block

    E, h, n, k, tokens, cap = 4, 256, 128, 2, 300, 384
    rng = np.random.default_rng(6)
    w = _weights(E, h, n, 7)
    x = rng.standard_normal((tokens, h)).astype(np.float32).astype(ml_dtypes.bfloat16)
    logits = rng.standard_normal((tokens, E)).astype(np.float32)
    ids, weights = R.route(logits, k)
    weights = weights.astype(np.float32).astype(np.float64)
    layer = MegaMoEFp8Block(*(T(v) for v in w), topk=k, max_tokens=tokens, rows_cap=cap)
    guards = []
    for name, cols, dtype, fill in (("a_q", h, torch.uint8, 0x7f), ("row_weight", 0, torch.float32, torch.nan), ("row_token", 0, torch.int32, -9),
                                    ("gateup", 2 * n, torch.bfloat16, torch.nan), ("d_q", n, torch.uint8, 0x7f), ("y", h, torch.bfloat16, torch.nan)):
        whole, part = _guarded(cap, cols, dtype, fill)
        setattr(layer, name, part)
        guards.append((name, whole[cap:], whole[cap:].clone()))
    tx, tl = T(x.view(np.int16)).view(torch.bfloat16), T(logits)
    got = layer.forward(tx, tl)
    assert _lib.status_word() == 0x00E00000
    for name, now, before in guards:
        assert torch.equal(now.view(torch.uint8), before.view(torch.uint8)), name
    want = _layer(x.astype(np.float32), _in_rows_cap(ids, 0, E, cap), weights, w)
    scale = np.abs(want).max()
    assert np.abs(got.double().cpu().numpy() - want).max() < 3e-2 * scale
    layer = MegaMoEFp8Block(*(T(v) for v in w), topk=k, max_tokens=tokens)
    _close(layer.forward(tx, tl).double().cpu().numpy(), _layer(x.astype(np.float32), ids, weights, w))


def test_a_small_rows_cap_of_the_nvfp4_layer():
    from mosaicist_b200 import _lib, ops
    from mosaicist_b200.moe import MegaMoE, RouteConfig

    E, h, n, k, cap = 4, 256, 256, 2, 384
    g = torch.Generator(device="cuda").manual_seed(0)
    w1, w2 = (0.05 * torch.randn(s, device="cuda", generator=g) for s in ((E, 2 * n, h), (E, h, n)))
    ones = torch.ones(E, device="cuda")
    gs1, gs2 = ops.global_scale_for(w1), ops.global_scale_for(w2)
    args = (*ops.quantize_nvfp4(w1, gs1), gs1, ones, *ops.quantize_nvfp4(w2, gs2), gs2, ones, 300 * ones, 300 * ones)
    for tokens in (300, 2500):                                 # scales written in place, and staged by rows
        x, logits = torch.randn(tokens, h, device="cuda", generator=g).bfloat16(), torch.randn(tokens, E, device="cuda", generator=g)
        small = MegaMoE(*args, topk=k, max_tokens=tokens, rows_cap=cap, route=RouteConfig())
        guards = []
        for name, cols, dtype, fill in (("a_q", h // 2, torch.uint8, 0x77), ("row_weight", 0, torch.float32, torch.nan),
                                        ("row_token", 0, torch.int32, -9), ("sf_rows", h // 16, torch.uint8, 0x7f), ("y", h, torch.bfloat16, torch.nan)):
            whole, part = _guarded(cap, cols, dtype, fill)
            setattr(small, name, part)
            guards.append((name, whole[cap:], whole[cap:].clone()))
        got = small.forward(x, logits)
        assert _lib.status_word() == 0x00E00000
        for name, now, before in guards:
            assert torch.equal(now.view(torch.uint8), before.view(torch.uint8)), name
        full = MegaMoE(*args, topk=k, max_tokens=tokens, route=RouteConfig())
        full.route(logits)
        full.ids[:tokens] = T(_in_rows_cap(full.ids[:tokens].cpu().numpy(), 0, E, cap))
        want = full.forward(x)
        assert _lib.status_word() == 0
        assert (got.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
        assert (want != 0).any()


@pytest.mark.parametrize("h", [23584, 23808, 24576])
def test_dispatch_of_rows_that_nearly_fill_the_default_shared_memory(h):
    """Two rows of 23584 to 23824 columns are under 48 KB, with the kernel's own arrays they are not."""
    test_dispatch_bit_exact(3, h, 8, 2, 0, 8)
