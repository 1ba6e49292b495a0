"""Refusals of the routing and FP8 block operators: by the host path on FakeTensors (device and shape, no
memory) and by the C ABI itself, which refuses before anything is launched.  No GPU work happens here."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mosaicist_b200 import _lib, ops

BF16, F16, F32, U8, I32, E4 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int32, torch.float8_e4m3fn


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield


def _t(*shape, dtype=F32, device="cuda"):
    return torch.empty(shape, dtype=dtype, device=device)


def _refused(call, *args):
    for a in args:
        with pytest.raises(ValueError):
            call(a)


def test_route_arguments(fake):
    x = _t(16, 64)
    _refused(lambda v: ops.moe_route(v, 4), _t(16, 64, device="cpu"), _t(16, 64, dtype=torch.float64), _t(64, 16).t(), _t(64),
             _t(2, 16, 64))
    _refused(lambda v: ops.moe_route(x, v), 0, -1, 65)
    _refused(lambda v: ops.moe_route(x, 4, bias=v), _t(63), _t(64, dtype=BF16), _t(64, device="cpu"), _t(1, 64), _t(128)[::2])
    _refused(lambda v: ops.moe_route(x, 4, score=v), "tanh", None, 0)
    _refused(lambda v: ops.moe_route(x, 4, groups=v), -1)
    ids, w = _t(16, 4, dtype=I32), _t(16, 4)
    _refused(lambda v: ops.moe_route(x, 4, out=v), (_t(16, 3, dtype=I32), w), (_t(16, 4, dtype=torch.int64), w), (ids, _t(16, 4, dtype=BF16)),
             (ids, _t(4, 16).t()), (ids,), (ids.cpu(), w))
    _refused(lambda v: ops.moe_route(x, 4, out=v), (ids, _t(16, 4, device="cuda:1")))


def test_route_backward_arguments(fake):
    g, x, ids, w = _t(16, 4), _t(16, 64), _t(16, 4, dtype=I32), _t(16, 4)
    _refused(lambda v: ops.moe_route_backward(v, x, ids, w), _t(16, 3), _t(15, 4), _t(16, 4, dtype=BF16), _t(4, 16).t(), _t(16, 4, device="cpu"))
    _refused(lambda v: ops.moe_route_backward(g, v, ids, w), _t(15, 64), _t(16, 64, dtype=torch.float64), _t(64, 16).t(), _t(16))
    _refused(lambda v: ops.moe_route_backward(g, x, v, w), _t(16, 4, dtype=torch.int64), _t(16, 3, dtype=I32), _t(16, dtype=I32))
    _refused(lambda v: ops.moe_route_backward(g, x, ids, v), _t(16, 3), _t(16, 4, dtype=F16))
    _refused(lambda v: ops.moe_route_backward(g, x, ids, w, out=v), _t(16, 63), _t(16, 64, dtype=BF16), _t(64, 16).t())
    _refused(lambda v: ops.moe_route_backward(g, x, ids, w, score=v), "none")


def test_quantizer_arguments(fake):
    x = _t(100, 272, dtype=BF16)
    q, sf = _t(100, 272, dtype=U8), _t(3, 100)
    _refused(lambda v: ops.quantize_fp8_block(v), x.cpu(), _t(272, 100).t(), _t(100), _t(100, 272, dtype=U8), _t(4, 100, 272))
    _refused(lambda v: ops.quantize_fp8_block(v, silu=True), _t(100, 271))
    _refused(lambda v: ops.quantize_fp8_block(x, out=v), (q[:99], sf), (q, _t(2, 100)), (q, _t(3, 104)), (q, _t(3, 100, dtype=BF16)),
             (_t(100, 272, dtype=BF16), sf), (q,), (q, _t(100, 3).t()))
    offs, rows = _t(4, dtype=I32), _t(4, dtype=I32)
    _refused(lambda v: ops.quantize_fp8_block(x, group_offsets=v, group_rows=rows), None, _t(3, dtype=I32), _t(4, dtype=torch.int64), _t(4, 1, dtype=I32))
    _refused(lambda v: ops.quantize_fp8_block(x, group_offsets=offs, group_rows=v), None, _t(5, dtype=I32), offs.cpu())
    _refused(lambda v: ops.quantize_fp8_block(x, group_offsets=v, group_rows=v), _t(0, dtype=I32))
    w = _t(260, 272)
    _refused(lambda v: ops.quantize_fp8_block_weight(v), w.cpu(), w.t(), _t(260), _t(1, 2, 260, 272), _t(260, 272, dtype=torch.float64))
    wq, wsf = _t(260, 272, dtype=U8), _t(3, 3)
    _refused(lambda v: ops.quantize_fp8_block_weight(w, out=v), (wq, _t(2, 3)), (wq[:259], wsf), (wq, _t(1, 3, 3)), (wq, wsf.cpu()))


def test_product_arguments(fake):
    a, sa, b, sb = _t(50, 272, dtype=U8), _t(3, 52), _t(264, 272, dtype=E4), _t(3, 3)
    call = ops.gemm_fp8_block
    _refused(lambda v: call(v, sa, b, sb), _t(50, 256, dtype=U8), _t(50, 272, dtype=BF16), a.cpu(), _t(272, 50, dtype=U8).t(), _t(272, dtype=U8))
    _refused(lambda v: call(a, v, b, sb), _t(3, 50), _t(52, 3).t(), _t(2, 52), _t(3, 52, dtype=BF16))
    _refused(lambda v: call(a, sa, v, sb), _t(264, 256, dtype=U8), _t(1, 264, 272, dtype=U8), _t(272, 264, dtype=U8).t())
    _refused(lambda v: call(a, sa, b, v), _t(2, 3), _t(3, 2), _t(3, 3, dtype=F16), _t(1, 3, 3))
    _refused(lambda v: call(a, sa, b, sb, out=v), _t(50, 263), _t(50, 264, dtype=U8), _t(264, 50).t(), _t(50, 264, device="cpu"))
    _refused(lambda v: call(a, sa, b, sb, out_dtype=v), torch.float64, U8, "bf16")
    _refused(lambda v: call(a, sa, b, sb, out_dtype=BF16, out=v), _t(50, 264))
    _refused(lambda v: call(a, sa, b, sb, max_ctas=v), -1)
    b3, sb3, offs, rows = _t(4, 264, 272, dtype=U8), _t(4, 3, 3), _t(4, dtype=I32), _t(4, dtype=I32)
    g = ops.ragged_grouped_gemm_fp8_block
    _refused(lambda v: g(a, sa, v, sb3, offs, rows), b, _t(3, 264, 272, dtype=U8), _t(4, 264, 288, dtype=U8))
    _refused(lambda v: g(a, sa, b3, v, offs, rows), sb, _t(3, 3, 3))
    _refused(lambda v: g(a, sa, b3, sb3, v, rows), _t(3, dtype=I32), _t(4, dtype=torch.int64), _t(4, dtype=I32, device="cpu"))
    _refused(lambda v: g(a, sa, b3, sb3, offs, v), _t(3, dtype=I32), _t(8, dtype=I32)[::2])
    _refused(lambda v: g(a, sa, b3, sb3, offs, rows, v), _t(49), _t(50, dtype=BF16), _t(50, 1))
    for arg in (sa, b3, sb3, offs, rows):
        args = [a, sa, b3, sb3, offs, rows]
        i = next(j for j, v in enumerate(args) if v is arg)
        args[i] = _t(*arg.shape, dtype=arg.dtype, device="cuda:1")
        with pytest.raises(ValueError, match="expected cuda:0"):
            g(*args)


# ---- the C ABI -----------------------------------------------------------------------------

P = 4096      # a pointer that nothing follows: the calls below are refused


@pytest.fixture(scope="module")
def lib():
    from mosaicist_b200 import build

    build.build()
    return _lib.load()


def _cfg(score=0, groups=1, topk_groups=1, group_top=1, renormalize=1, scale=1.0):
    return _lib.RouteCfg(score, groups, topk_groups, group_top, renormalize, scale)


def _route(lib, logits=P, dtype=1, bias=None, ids=P, w=P, tokens=8, experts=64, topk=4, cfg=None):
    return lib.msc_moe_route(logits, dtype, bias, ids, w, tokens, experts, topk, ctypes.byref(cfg or _cfg()), None)


@pytest.mark.parametrize("kw", [
    dict(logits=None), dict(ids=None), dict(w=None), dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(experts=0), dict(experts=1025),
    dict(topk=0), dict(topk=33), dict(topk=65), dict(logits=P + 2), dict(logits=P + 1, dtype=0), dict(bias=P + 2), dict(ids=P + 1), dict(w=P + 2),
    dict(cfg=_cfg(score=2)), dict(cfg=_cfg(groups=0)), dict(cfg=_cfg(groups=3)), dict(cfg=_cfg(groups=64)), dict(cfg=_cfg(groups=8, topk_groups=0)),
    dict(cfg=_cfg(groups=8, topk_groups=9)), dict(cfg=_cfg(group_top=0)), dict(cfg=_cfg(group_top=3)),
    dict(cfg=_cfg(groups=32, group_top=2), experts=32), dict(cfg=_cfg(groups=16, topk_groups=1), topk=5), dict(cfg=_cfg(scale=0.0)),
    dict(cfg=_cfg(scale=-1.0)), dict(cfg=_cfg(scale=float("nan"))), dict(cfg=_cfg(scale=float("inf"))),
    dict(cfg=_cfg(groups=31, topk_groups=4), experts=31 * 33), dict(cfg=_cfg(groups=20, topk_groups=4), experts=20 * 40)])
def test_route_refusals(lib, kw):
    assert _route(lib, **kw) in (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)
    assert lib.msc_last_error()


def test_empty_calls_do_nothing(lib):
    assert _route(lib, tokens=0) == _lib.OK
    assert lib.msc_moe_route_backward(P, P, 1, P, P, P, 0, 64, 4, 0, 1, 1.0, None) == _lib.OK
    assert lib.msc_fp8_block_quantize(P, 0, 0, None, None, P, P, 0, 0, 128, None) == _lib.OK
    assert lib.msc_gemm_fp8_block(P, P, P, P, P, 0, 0, 128, 128, 0, None) == _lib.OK


@pytest.mark.parametrize("args", [
    (None, P, 1, P, P, P, 8, 64, 4, 0, 1, 1.0), (P, None, 1, P, P, P, 8, 64, 4, 0, 1, 1.0), (P, P, 1, None, P, P, 8, 64, 4, 0, 1, 1.0),
    (P, P, 1, P, None, P, 8, 64, 4, 0, 1, 1.0), (P, P, 1, P, P, None, 8, 64, 4, 0, 1, 1.0), (P, P, 5, P, P, P, 8, 64, 4, 0, 1, 1.0),
    (P, P, 1, P, P, P, -8, 64, 4, 0, 1, 1.0), (P, P, 1, P, P, P, 8, 2000, 4, 0, 1, 1.0), (P, P, 1, P, P, P, 8, 64, 40, 0, 1, 1.0),
    (P, P, 1, P, P, P, 8, 64, 4, 2, 1, 1.0), (P, P, 1, P, P, P, 8, 64, 4, 0, 1, 0.0), (P + 1, P, 1, P, P, P, 8, 64, 4, 0, 1, 1.0),
    (P, P, 1, P, P, P + 2, 8, 64, 4, 0, 1, 1.0)])
def test_route_backward_refusals(lib, args):
    assert lib.msc_moe_route_backward(*args, None) in (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)


@pytest.mark.parametrize("args", [
    (None, 0, 0, None, None, P, P, 0, 8, 128), (P, 0, 0, None, None, None, P, 0, 8, 128), (P, 0, 0, None, None, P, None, 0, 8, 128),
    (P, 0, 0, P, None, P, P, 1, 8, 128), (P, 0, 0, None, P, P, P, 1, 8, 128), (P, 0, 0, P, P, P, P, 0, 8, 128), (P, 0, 0, None, None, P, P, 0, -1, 128),
    (P, 0, 0, None, None, P, P, 0, 8, 0), (P, 0, 0, None, None, P, P, 0, 8, 120), (P, 3, 0, None, None, P, P, 0, 8, 128),
    (P + 8, 0, 0, None, None, P, P, 0, 8, 128), (P, 0, 0, None, None, P + 8, P, 0, 8, 128), (P, 0, 0, None, None, P, P + 2, 0, 8, 128),
    (P, 0, 0, None, None, P, P, 0, 0x7fffffff, 128), (P, 0, 0, None, None, P, P, 0, 8, 0x7ffffff0)])
def test_quantizer_refusals(lib, args):
    assert lib.msc_fp8_block_quantize(*args, None) in (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)


@pytest.mark.parametrize("args", [
    (None, 0, P, P, 1, 128, 128), (P, 0, None, P, 1, 128, 128), (P, 0, P, None, 1, 128, 128), (P, 0, P, P, 0, 128, 128), (P, 0, P, P, 1, 0, 128),
    (P, 0, P, P, 1, 128, 0), (P, 0, P, P, 1, 128, 100), (P, 7, P, P, 1, 128, 128), (P + 4, 0, P, P, 1, 128, 128), (P, 0, P + 4, P, 1, 128, 128),
    (P, 0, P, P + 1, 1, 128, 128), (P, 0, P, P, 70000, 128, 128), (P, 0, P, P, 1, 0x7fffffff, 128), (P, 0, P, P, 1, 128, 0x7ffffff0)])
def test_weight_quantizer_refusals(lib, args):
    assert lib.msc_fp8_block_quantize_weight(*args, None) in (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)


@pytest.mark.parametrize("args", [
    (None, P, P, P, P, 0, 8, 128, 128, 0), (P, None, P, P, P, 0, 8, 128, 128, 0), (P, P, None, P, P, 0, 8, 128, 128, 0),
    (P, P, P, None, P, 0, 8, 128, 128, 0), (P, P, P, P, None, 0, 8, 128, 128, 0), (P, P, P, P, P, 3, 8, 128, 128, 0),
    (P, P, P, P, P, 0, -1, 128, 128, 0), (P, P, P, P, P, 0, 8, 0, 128, 0), (P, P, P, P, P, 0, 8, 128, 0, 0), (P, P, P, P, P, 0, 8, 100, 128, 0),
    (P, P, P, P, P, 0, 8, 128, 100, 0), (P, P, P, P, P, 0, 8, 128, 128, -2), (P + 8, P, P, P, P, 0, 8, 128, 128, 0), (P, P + 4, P, P, P, 0, 8, 128, 128, 0),
    (P, P, P + 1, P, P, 0, 8, 128, 128, 0), (P, P, P, P + 2, P, 0, 8, 128, 128, 0), (P, P, P, P, P + 8, 0, 8, 128, 128, 0),
    (P, P, P, P, P, 0, 0x7fffffff, 128, 128, 0), (P, P, P, P, P, 0, 8, 0x7ffffff8, 128, 0), (P, P, P, P, P, 0, 8, 128, 0x7ffffff0, 0)])
def test_product_refusals(lib, args):
    assert lib.msc_gemm_fp8_block(*args, None) in (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)


@pytest.mark.parametrize("args", [
    (P, P, P, P, None, P, None, P, 0, 2, 8, 128, 128, 0), (P, P, P, P, P, None, None, P, 0, 2, 8, 128, 128, 0), (P, P, P, P, P, P, None, P, 0, 0, 8, 128, 128, 0),
    (P, P, P, P, P, P, P + 2, P, 0, 2, 8, 128, 128, 0), (P, P, P, P, P, P, None, P, 0, 1 << 20, 8, 1 << 12, 128, 0)])
def test_grouped_product_refusals(lib, args):
    assert lib.msc_grouped_gemm_fp8_block_ragged(*args, None) in (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)


def test_operators_can_be_traced(fake):
    import mosaicist_b200.torch_ops as O

    x = _t(10, 544, dtype=BF16)
    q, sf = O.quantize_fp8_block(x, True, None, None)
    assert q.shape == (10, 272) and sf.shape == (3, 12) and sf.dtype == F32
    wq, wsf = O.quantize_fp8_block_weight(_t(2, 136, 272))
    assert wq.shape == (2, 136, 272) and wsf.shape == (2, 2, 3)
    assert O.gemm_fp8_block(q, sf, wq[0], wsf[0], F16).dtype == F16
    assert O.grouped_gemm_fp8_block_ragged(q, sf, wq, wsf, _t(2, dtype=I32), _t(2, dtype=I32), None, F32).shape == (10, 136)
    ids, w = O.moe_route(_t(10, 64), 4, "sigmoid", None, 1, 1, 1, True, 1.0)
    assert ids.dtype == I32 and w.shape == (10, 4)
    assert O.moe_route_backward(w, _t(10, 64, dtype=F16), ids, w, "sigmoid", True, 1.0).dtype == F16


@pytest.mark.parametrize("kw", [
    dict(tokens_ptr=None), dict(ids=None), dict(w=None), dict(rank=None), dict(offs=None), dict(a_q=None), dict(a_sf=None), dict(rw=None), dict(rt=None),
    dict(tokens=-1), dict(hidden=0), dict(hidden=100), dict(topk=0), dict(topk=65), dict(local=0), dict(cap=0), dict(tokens_ptr=P + 2), dict(a_q=P + 8),
    dict(a_sf=P + 2), dict(ids=P + 1), dict(hidden=200000), dict(hidden=0x7ffffff0), dict(cap=0x7fffffff)])
def test_dispatch_refusals(lib, kw):
    a = dict(tokens_ptr=P, ids=P, w=P, rank=P, offs=P, tokens=8, hidden=256, topk=2, first=0, local=4, a_q=P, a_sf=P, rw=P, rt=P, cap=512) | kw
    assert lib.msc_moe_permute_quantize_fp8_block(*a.values(), None) in (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)


def _layer_stub(**kw):
    from types import SimpleNamespace

    T, K, E, h, cap = 16, 2, 8, 272, 1152
    i32 = lambda *s: _t(*s, dtype=I32)
    return SimpleNamespace(**(dict(
        ids=i32(T, K), weights=_t(T, K), rank=i32(T, K), group_rows=i32(E), group_offsets=i32(E), total_rows=i32(1), scratch=i32(4), topk=K, E=E,
        expert_first=0, h=h, a_q=_t(cap, h, dtype=U8), a_sf=_t(3, cap), row_weight=_t(cap), row_token=i32(cap), rows_cap=cap) | kw))


def test_fp8_layer_buffers(fake):
    from mosaicist_b200.moe import _host_ops

    x = _t(16, 272, dtype=BF16)
    for kw in (dict(ids=_t(15, 2, dtype=I32)), dict(weights=_t(16, 2, dtype=BF16)), dict(rank=_t(16, 1, dtype=I32)), dict(a_q=_t(1151, 272, dtype=U8)),
               dict(a_sf=_t(2, 1152)), dict(a_sf=_t(3, 1148)), dict(row_weight=_t(1151)), dict(row_token=_t(1152)), dict(group_rows=_t(7, dtype=I32)),
               dict(a_q=_t(1152, 272, dtype=U8, device="cuda:1")), dict(row_weight=None)):
        with pytest.raises(ValueError):
            _host_ops.moe_dispatch_fp8_block(_layer_stub(**kw), x)
    for bad in (_t(17, 272, dtype=BF16), _t(16, 256, dtype=BF16), _t(16, 272), _t(16, 272, dtype=BF16, device="cpu"), _t(272, 16, dtype=BF16).t()):
        with pytest.raises(ValueError):
            _host_ops.moe_dispatch_fp8_block(_layer_stub(), bad)


def test_fp8_layer_arguments(fake):
    from mosaicist_b200.moe import MegaMoEFp8Block

    w1, s1, w2, s2 = _t(4, 512, 256, dtype=U8), _t(4, 4, 2), _t(4, 256, 256, dtype=U8), _t(4, 2, 2)
    layer = MegaMoEFp8Block(w1, s1, w2, s2, topk=2, max_tokens=8)
    assert layer.rows_cap == 640 and layer.a_sf.shape == (2, 640)
    for kw in (dict(topk=0), dict(topk=33), dict(max_tokens=0), dict(rows_cap=100), dict(rows_cap=0)):
        with pytest.raises(ValueError):
            MegaMoEFp8Block(w1, s1, w2, s2, **(dict(topk=2, max_tokens=8) | kw))
    for a, b in ((w1[0], w2), (w1, w2[:3]), (w1[:, :511], w2), (_t(4, 512, 248, dtype=U8), _t(4, 248, 256, dtype=U8)), (w1, _t(4, 256, 128, dtype=U8))):
        with pytest.raises(ValueError):
            MegaMoEFp8Block(a, s1, b, s2, topk=2, max_tokens=8)
    for call in (lambda: layer.forward(_t(9, 256, dtype=BF16)), lambda: layer.route(_t(9, 4)), lambda: layer.forward(_t(8, 256, dtype=BF16), _t(7, 4))):
        with pytest.raises(ValueError):
            call()


def test_fp8_layer_without_a_router_of_its_own(fake, monkeypatch):
    """route=None is the plain rule, as MegaMoE has it."""
    from mosaicist_b200 import moe

    w1, s1, w2, s2 = _t(4, 512, 256, dtype=U8), _t(4, 4, 2), _t(4, 256, 256, dtype=U8), _t(4, 2, 2)
    seen = []
    monkeypatch.setattr(ops, "moe_route", lambda *args: seen.append(args[1:9]))
    for kw in (dict(), dict(route=None), dict(route=moe.RouteConfig())):
        moe.MegaMoEFp8Block(w1, s1, w2, s2, topk=2, max_tokens=8, **kw).route(_t(8, 4))
    assert seen == [(2, "softmax", None, 1, 1, 1, True, 1.0)] * 3


def test_empty_calls_check_their_arguments(lib):
    """Nothing to do is no reason to take a wrong configuration; what is empty needs no memory."""
    bad = (_lib.ERR_BAD_ARG, _lib.ERR_UNSUPPORTED)
    none = dict(logits=None, ids=None, w=None, tokens=0)
    assert _route(lib, **none) == _lib.OK
    for cfg in (_cfg(score=2), _cfg(groups=3), _cfg(groups=8, topk_groups=9), _cfg(scale=0.0)):
        assert _route(lib, cfg=cfg, **none) in bad
    assert _route(lib, topk=65, **none) in bad
    back = lambda *a: lib.msc_moe_route_backward(None, None, 1, None, None, None, 0, *a, None)
    assert back(64, 4, 0, 1, 1.0) == _lib.OK and back(64, 4, 2, 1, 1.0) in bad and back(64, 4, 0, 1, -1.0) in bad and back(64, 0, 0, 1, 1.0) in bad
    quant = lambda *a: lib.msc_fp8_block_quantize(None, *a, None)
    assert quant(0, 0, None, None, None, None, 0, 0, 128) == _lib.OK and quant(0, 0, None, None, None, None, 0, 0, 100) in bad
    gemm = lambda *a: lib.msc_gemm_fp8_block(None, None, P, P, None, *a, None)
    assert gemm(0, 0, 128, 128, 0) == _lib.OK and gemm(0, 0, 100, 128, 0) in bad and gemm(0, 0, 128, 100, 0) in bad and gemm(5, 0, 128, 128, 0) in bad
