"""The peer-memory expert-parallel exchange on ONE device: several ranks' layers live in one
process, every phase runs for all of them before the next phase starts (which is what the
barriers guarantee between real ranks), and the buffers a rank would reach over NVLink are
plain tensors of the same device.  Each rank's output must equal, bit for bit, what the
single-GPU layer computes for the same tokens; the placement kernel must equal its oracle."""

import ml_dtypes
import numpy as np
import pytest
import torch

from oracle import moe as M
from tests.test_moe_gpu import T, _dev_weights, _weights

pytestmark = pytest.mark.gpu


def _layers(world, E, k, h, n, T_loc, rows_cap, w, input_gs, a2_gs, push=False, flags=False, presum=False):
    from mosaicist_b200.moe import MegaMoE
    from mosaicist_b200.parallel import EXCHANGE_BUFFERS, PeerExpertParallelMoE, exchange_layout, exchange_views

    el = E // world
    d = _dev_weights(w)
    pairs_cap = T_loc * k if push else 0
    _, total = exchange_layout(rows_cap, h, pairs_cap, world, E)
    spaces = [exchange_views(torch.zeros(total, dtype=torch.uint8, device="cuda"), rows_cap, h, pairs_cap, world, E)
              for _ in range(world)]
    pointers = {name: [s[name].data_ptr() for s in spaces] for name in EXCHANGE_BUFFERS}
    ranks = []
    for r in range(world):
        sl = slice(r * el, (r + 1) * el)
        layer = MegaMoE(d["w1_q"][sl], d["w1_sf"][sl], d["w1_gs"][sl], d["w1_alpha"][sl], d["w2_q"][sl],
                        d["w2_sf"][sl], d["w2_gs"][sl], d["w2_alpha"][sl], T(input_gs[sl]), T(a2_gs[sl]),
                        topk=1, max_tokens=1, expert_first=r * el, rows_cap=rows_cap, workspace=spaces[r])
        extra = dict(row_dest=spaces[r]["row_dest"], recv_y=spaces[r]["recv_y"]) if push else {}
        if flags:
            extra.update(flags=spaces[r]["flags"], counts_all=spaces[r]["counts_all"])
        if presum:
            extra.update(row_next=spaces[r]["row_next"])
        ranks.append(PeerExpertParallelMoE(layer, pointers, spaces[r]["sf_rows"], T(input_gs), E, k, T_loc, r,
                                           world, **extra))
    return ranks


def _lockstep(ranks, tokens, logits):
    """One layer call of every rank, phase by phase.  With flag synchronisation every rank's
    signal of a phase is launched before any rank's wait for it, so no wait ever spins."""
    from mosaicist_b200.parallel import SLOT_COUNTS, SLOT_RESULTS_READY, SLOT_ROWS_LANDED

    flags = ranks[0].flag_sync
    for ep, lg in zip(ranks, logits):
        ep.count(lg)
    if flags:
        for ep in ranks:
            ep.epoch += 1
            ep.signal(SLOT_COUNTS, with_counts=True)
        for ep in ranks:
            ep.place(wait=True)
        counts_all = ranks[0].counts_all.clone()
    else:
        counts_all = torch.stack([ep.counts for ep in ranks]).contiguous()
        for ep in ranks:
            ep.place(counts_all)
    for ep, tk in zip(ranks, tokens):
        ep.dispatch(tk)
    if flags:
        for ep in ranks:
            ep.signal(SLOT_ROWS_LANDED)
        for ep in ranks:
            ep.wait(SLOT_ROWS_LANDED)
    for ep in ranks:
        ep.experts()
    if flags:
        for ep in ranks:
            ep.signal(SLOT_RESULTS_READY)
        for ep in ranks:
            ep.wait(SLOT_RESULTS_READY)
    return [ep.combine() for ep in ranks], counts_all


@pytest.mark.parametrize("flags", [False, True], ids=["collectives", "flags"])
@pytest.mark.parametrize("push", [False, True], ids=["pull", "push"])
@pytest.mark.parametrize("world,E,k,h,n,T_loc", [(2, 32, 2, 256, 128, 160), (4, 32, 4, 512, 256, 96),
                                                  (8, 64, 8, 256, 128, 40),
                                                  (2, 32, 3, 384, 128, 70)])   # h % 256 != 0: store dispatch
def test_emulated_ranks_equal_single_gpu_layer(world, E, k, h, n, T_loc, push, flags):
    if push and h % 256:
        pytest.skip("the row-scatter GEMM needs n % 256 == 0")
    from mosaicist_b200 import _lib
    from mosaicist_b200.moe import MegaMoE

    w = _weights(E, h, n, seed=world)
    rng = np.random.default_rng([world, 9])
    tokens = [rng.standard_normal((T_loc, h)).astype(np.float32).astype(ml_dtypes.bfloat16) for _ in range(world)]
    logits = [rng.standard_normal((T_loc, E)).astype(np.float32) for _ in range(world)]
    # two distinct input scales, so that a token block is requantised between its experts
    input_gs = np.where(np.arange(E) % 3 == 0, 2688.0 / 4.0, 2688.0 / 5.0).astype(np.float32)
    a2_gs = np.full(E, 2688.0 / 4.0, np.float32)
    rows_cap = (world * T_loc * k + 127 * (E // world) + 127) // 128 * 128
    ranks = _layers(world, E, k, h, n, T_loc, rows_cap, w, input_gs, a2_gs, push, flags)
    tk = [T(np.asarray(t, np.float32)).to(torch.bfloat16) for t in tokens]
    lg = [T(l) for l in logits]
    for _ in range(2):                                     # buffers are reusable as they are
        outs, counts_all = _lockstep(ranks, tk, lg)
    assert _lib.status_word() == 0

    # placement kernel == oracle
    ca = counts_all.cpu().numpy()
    for r, ep in enumerate(ranks):
        ids, _ = M.route_topk(logits[r], k)
        _, counts, _, _ = M.plan(ids, 0, E)
        assert np.array_equal(ca[r], counts)
        send_base, rows, offs, total = M.ep_placement(ca, r)
        assert np.array_equal(ep.send_base.cpu().numpy(), send_base)
        assert np.array_equal(ep.layer.group_rows.cpu().numpy(), rows)
        assert np.array_equal(ep.layer.group_offsets.cpu().numpy(), offs)
        assert int(ep.layer.total_rows[0]) == total

    # every rank's output == the single-GPU layer over all experts on that rank's tokens
    d = _dev_weights(w)
    single = MegaMoE(d["w1_q"], d["w1_sf"], d["w1_gs"], d["w1_alpha"], d["w2_q"], d["w2_sf"], d["w2_gs"],
                     d["w2_alpha"], T(input_gs), T(a2_gs), topk=k, max_tokens=T_loc)
    for r in range(world):
        want = single.forward(tk[r], lg[r])
        assert torch.equal(outs[r], want), (r, (outs[r].float() - want.float()).abs().max())
        assert np.count_nonzero(want.float().cpu().numpy()) > 0.9 * want.numel()
    assert _lib.status_word() == 0


@pytest.mark.parametrize("world,E,k,h,n,T_loc", [(2, 32, 4, 256, 128, 160), (4, 32, 8, 512, 256, 96)])
def test_presummed_combine_is_within_tolerance_and_sends_fewer_rows(world, E, k, h, n, T_loc):
    """A token's result rows that live on one rank are summed there (fp32, pair order, one bf16
    rounding) before they are sent: every (token, rank) pair delivers exactly one row, the pairs
    absorbed into it are marked -2, and the layer output stays within the MoE bound of the
    reference's tests (test_kernels.py:94-102: max-rel < 1e-1, rms-rel < 1e-2) of the
    single-GPU layer - it is no longer bit-identical, the partial sums are rounded once more."""
    from mosaicist_b200 import _lib
    from mosaicist_b200.moe import MegaMoE

    w = _weights(E, h, n, seed=world + 20)
    rng = np.random.default_rng([world, 11])
    tokens = [rng.standard_normal((T_loc, h)).astype(np.float32).astype(ml_dtypes.bfloat16) for _ in range(world)]
    logits = [rng.standard_normal((T_loc, E)).astype(np.float32) for _ in range(world)]
    input_gs = np.full(E, 2688.0 / 5.0, np.float32)
    a2_gs = np.full(E, 2688.0 / 4.0, np.float32)
    rows_cap = (world * T_loc * k + 127 * (E // world) + 127) // 128 * 128
    ranks = _layers(world, E, k, h, n, T_loc, rows_cap, w, input_gs, a2_gs, push=True, presum=True)
    tk = [T(np.asarray(t, np.float32)).to(torch.bfloat16) for t in tokens]
    lg = [T(l) for l in logits]
    for _ in range(2):
        outs, _ = _lockstep(ranks, tk, lg)
    assert _lib.status_word() == 0
    d = _dev_weights(w)
    single = MegaMoE(d["w1_q"], d["w1_sf"], d["w1_gs"], d["w1_alpha"], d["w2_q"], d["w2_sf"], d["w2_gs"],
                     d["w2_alpha"], T(input_gs), T(a2_gs), topk=k, max_tokens=T_loc)
    el = E // world
    for r in range(world):
        want = single.forward(tk[r], lg[r]).float().cpu().numpy()
        got = outs[r].float().cpu().numpy()
        err = np.abs(got - want)
        assert err.max() <= 1e-1 * np.abs(want).max() and np.sqrt((err ** 2).mean()) <= 1e-2 * np.sqrt((want ** 2).mean())
        assert not np.array_equal(got, want) or k == 1
        # one delivered row per (token, owner rank); the rest of the token's pairs are absorbed
        ids, _ = M.route_topk(logits[r], k)
        owners = ids // el
        pr = ranks[r].pair_row[:T_loc].cpu().numpy()
        for t in range(T_loc):
            first = {o: int(np.flatnonzero(owners[t] == o)[0]) for o in set(owners[t].tolist())}
            for kk in range(k):
                assert (pr[t, kk] >= 0) == (first[owners[t, kk]] == kk)
                assert pr[t, kk] >= 0 or pr[t, kk] == -2
        assert (pr == -2).any()


def test_overflowing_rank_drops_rows_and_raises_the_status_bit():
    """More rows than rows_cap: nothing is stored out of bounds, the status word reports it."""
    from mosaicist_b200 import _lib

    world, E, k, h, n, T_loc = 2, 32, 2, 256, 128, 160
    w = _weights(E, h, n, seed=1)
    rng = np.random.default_rng(3)
    tokens = [T(rng.standard_normal((T_loc, h)).astype(np.float32)).to(torch.bfloat16) for _ in range(world)]
    logits = [T(rng.standard_normal((T_loc, E)).astype(np.float32)) for _ in range(world)]
    gs = np.full(E, 2688.0 / 5.0, np.float32)
    ranks = _layers(world, E, k, h, n, T_loc, 128, w, gs, gs)        # far too small
    for ep, lg in zip(ranks, logits):
        ep.count(lg)
    counts_all = torch.stack([ep.counts for ep in ranks]).contiguous()
    for ep, tk in zip(ranks, tokens):
        ep.place(counts_all)
        ep.dispatch(tk)
    assert _lib.status_word() & 0x00E00000
    ca = counts_all.cpu().numpy()
    for r, ep in enumerate(ranks):
        rows = ep.pair_row[:T_loc].cpu().numpy()
        ids = ep.ids[:T_loc].cpu().numpy()
        dest = M.ep_placement(ca, r)[0][ids] + ep.rank_in_group[:T_loc].cpu().numpy()
        assert np.array_equal(rows, np.where(dest < 128, dest, -1))     # dropped pairs are marked
        assert (rows == -1).any()


def test_overflowing_push_layer_stays_inside_its_buffers_and_skips_dropped_pairs():
    """The whole pushed layer with rows_cap far too small: the group tables are cut to rows_cap,
    the GEMMs and the scatter stay inside the buffers, pairs that did not fit are left out of the
    sum (their recv_y rows are pre-filled with NaN here, standing in for an earlier step's
    data), and the status word says what happened."""
    from mosaicist_b200 import _lib

    world, E, k, h, n, T_loc = 2, 32, 2, 256, 128, 160
    w = _weights(E, h, n, seed=2)
    rng = np.random.default_rng(5)
    tokens = [T(rng.standard_normal((T_loc, h)).astype(np.float32)).to(torch.bfloat16) for _ in range(world)]
    logits = [T(rng.standard_normal((T_loc, E)).astype(np.float32)) for _ in range(world)]
    gs = np.full(E, 2688.0 / 5.0, np.float32)
    rows_cap = 256
    ranks = _layers(world, E, k, h, n, T_loc, rows_cap, w, gs, gs, push=True)
    for ep in ranks:
        ep.recv_y.fill_(float("nan"))
    outs, counts_all = _lockstep(ranks, tokens, logits)
    torch.cuda.synchronize()
    assert _lib.status_word() & 0x00E00000
    for r, ep in enumerate(ranks):
        assert int(ep.layer.total_rows[0]) <= rows_cap
        table_end = (ep.layer.group_offsets + ep.layer.group_rows).max()
        assert int(table_end) <= rows_cap
        rows = ep.pair_row[:T_loc]
        assert bool((rows < 0).any()) and bool((rows >= 0).any())
        assert not bool(torch.isnan(outs[r]).any()), "a dropped pair's stale row entered the sum"
        kept = (rows >= 0).any(dim=1)
        assert bool((outs[r][kept].float().abs().sum(dim=1) > 0).all())
        assert bool((outs[r][~kept] == 0).all())
        assert bool((ep.row_dest == -1).all())     # reset for the next step


def test_wait_without_signal_times_out_and_reports():
    """A flag nobody raises: the wait gives up after its limit, sets the status bit, and the
    context stays usable (the next kernel runs)."""
    import time

    from mosaicist_b200 import _lib

    lib = _lib.load()
    flags = torch.zeros(64, dtype=torch.int32, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    t0 = time.perf_counter()
    _lib.check(lib.msc_ep_wait(flags.data_ptr(), 2, 1, 1, st))
    torch.cuda.synchronize()
    took = time.perf_counter() - t0
    assert 0.5 < took < 10.0
    assert _lib.status_word() & 0x00D00000
    assert int((flags + 1).sum()) == 64          # the device still answers
    assert _lib.status_word() == 0


@pytest.mark.parametrize("push", [False, True], ids=["pull", "push"])
def test_emulated_ranks_route_by_the_layers_rule(push):
    from mosaicist_b200 import _lib, ops
    from mosaicist_b200.moe import MegaMoE, RouteConfig

    world, E, k, h, n, T_loc = 2, 32, 4, 256, 128, 60
    w = _weights(E, h, n, seed=3)
    rng = np.random.default_rng(4)
    cfg = RouteConfig(score="sigmoid", groups=4, topk_groups=2, group_top=2, scale=2.0)
    bias = T((0.2 * rng.standard_normal(E)).astype(np.float32))
    gs, gs2 = np.full(E, 2688.0 / 5.0, np.float32), np.full(E, 2688.0 / 4.0, np.float32)
    rows_cap = (world * T_loc * k + 127 * (E // world) + 127) // 128 * 128
    ranks = _layers(world, E, k, h, n, T_loc, rows_cap, w, gs, gs2, push)
    for ep in ranks:
        ep.layer.route_config, ep.layer.route_bias = cfg, bias
    tk = [T(rng.standard_normal((T_loc, h)).astype(np.float32)).to(torch.bfloat16) for _ in range(world)]
    lg = [T(rng.standard_normal((T_loc, E)).astype(np.float32)) for _ in range(world)]
    outs, _ = _lockstep(ranks, tk, lg)
    d = _dev_weights(w)
    single = MegaMoE(d["w1_q"], d["w1_sf"], d["w1_gs"], d["w1_alpha"], d["w2_q"], d["w2_sf"], d["w2_gs"], d["w2_alpha"],
                     T(gs), T(gs2), topk=k, max_tokens=T_loc, route=cfg, route_bias=bias)
    for r in range(world):
        ids, _ = ops.moe_route(lg[r], k, "sigmoid", bias, 4, 2, 2, True, 2.0)
        assert torch.equal(ranks[r].ids[:T_loc], ids)
        assert torch.equal(outs[r], single.forward(tk[r], lg[r]))
    assert _lib.status_word() == 0
