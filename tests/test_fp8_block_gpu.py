"""FP8 operators with fp32 scales per block of 128 against the oracle."""

import ml_dtypes
import numpy as np
import pytest
import torch

from oracle import fp8_block as F

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def T(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    from mosaicist_b200 import _lib

    assert _lib.status_word() == 0


# ---- quantisers ----------------------------------------------------------------------------


def _rows(rng, rows, k):
    x = rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, 1)))
    x[rng.integers(0, rows), :] = 0
    return x.astype(np.float32)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 128), (3, 144), (8, 512), (9, 528), (17, 1040), (130, 7168), (1000, 64)])
def test_quantize_rows(rows, k, dtype):
    from mosaicist_b200 import ops

    x = T(_rows(np.random.default_rng([rows, k]), rows, k)).to(DT[dtype])
    q, sf = ops.quantize_fp8_block(x)
    want_q, want_sf = F.quantize_rows(x.float().cpu().numpy())
    pitch = (rows + 3) // 4 * 4
    assert q.dtype == torch.uint8 and sf.shape == (-(-k // 128), pitch)
    assert np.array_equal(sf.cpu().numpy()[:, :rows], want_sf) and (sf[:, rows:] == 0).all()
    assert np.array_equal(q.cpu().numpy(), want_q)


def test_quantize_more_rows_than_a_grid_is_high():
    """The rows of 65536 tokens with 8 experts each, and a few."""
    rows, k = 65536 * 8 + 3, 32
    from mosaicist_b200 import ops

    x = torch.randn(rows, k, device="cuda", dtype=torch.bfloat16)
    q, sf = ops.quantize_fp8_block(x)
    part, part_sf = ops.quantize_fp8_block(x[-4:].contiguous())
    assert torch.equal(q[-4:].view(torch.uint8), part.view(torch.uint8)) and torch.equal(sf[:, rows - 4:rows], part_sf)
    assert float(sf[:, rows:].abs().sum()) == 0
    assert torch.equal(sf[0, :rows], (x.float().abs().amax(1).cpu() / 448.0).cuda())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(8, 16), (1, 128), (128, 128), (129, 144), (1048, 400), (3, 260, 272)])
def test_quantize_weight(shape, dtype):
    from mosaicist_b200 import ops

    rng = np.random.default_rng(shape)
    w = T((rng.standard_normal(shape) * 0.02).astype(np.float32)).to(DT[dtype])
    q, sf = ops.quantize_fp8_block_weight(w)
    mats = w.float().cpu().numpy().reshape(-1, *shape[-2:])
    for i, m in enumerate(mats):
        want_q, want_sf = F.quantize_weight(m)
        assert np.array_equal(q.cpu().numpy().reshape(mats.shape)[i], want_q)
        assert np.array_equal(sf.cpu().numpy().reshape(-1, *want_sf.shape)[i], want_sf)
    assert q.shape == w.shape and sf.dim() == w.dim()
    again = ops.quantize_fp8_block_weight(w, out=(torch.empty_like(q), torch.empty_like(sf)))
    assert torch.equal(again[0], q) and torch.equal(again[1], sf)


def test_quotients_at_the_rounding_borders():
    """Values within two fp32 steps of every border between e4m3 values, times scales of all sizes: the
    byte is that of the correctly rounded quotient."""
    from mosaicist_b200 import ops

    rng = np.random.default_rng(0)
    codes = np.arange(0, 127, dtype=np.uint8).view(ml_dtypes.float8_e4m3fn).astype(np.float64)
    borders = (codes[:-1] + codes[1:]) / 2
    rows = 20000
    amax = (2.0 ** rng.uniform(-90, 90, rows)).astype(np.float32)
    amax[:100] = (2.0 ** rng.uniform(-140, -80, 100)).astype(np.float32)      # where division itself is used
    amax[100:200] = (2.0 ** rng.uniform(90, 127, 100)).astype(np.float32)
    s = F.block_scale(amax)
    x = (borders[None, :] * s[:, None].astype(np.float64)).astype(np.float32)
    x = np.where(x > 0, (x.view(np.int32) + rng.integers(-2, 3, x.shape, dtype=np.int32)).view(np.float32), x)
    x = np.where(np.abs(x) < amax[:, None], x, 0) * rng.choice([-1, 1], x.shape).astype(np.float32)
    x = np.concatenate([amax[:, None], x, np.zeros((rows, 1), np.float32)], 1)
    q, sf = ops.quantize_fp8_block(T(x))
    want_q, want_sf = F.quantize_rows(x)
    assert np.array_equal(sf.cpu().numpy(), want_sf) and np.array_equal(q.cpu().numpy(), want_q)


def test_zeros_infinities_and_nans():
    from mosaicist_b200 import ops

    x = torch.randn(8, 256, device="cuda")
    x[0] = 0
    x[1, :128] = 1e-42
    x[2, 7] = torch.inf
    x[3, 200] = torch.nan
    x[4] = torch.nan
    x[5] = torch.finfo(torch.float32).max
    q, sf = ops.quantize_fp8_block(x)
    v = q.view(torch.float8_e4m3fn).float()
    tiny = 2.0 ** -126
    assert (v[0] == 0).all() and (sf[:, 0] == tiny).all() and sf[0, 1] == tiny and (v[1, :128] == 0).all()
    assert sf[0, 2] == torch.inf and v[2, 7].isnan() and (v[2, :7] == 0).all() and sf[1, 2].isfinite()
    assert v[3, 200].isnan() and v[3].isnan().sum() == 1
    # (numpy's quotient: torch on a GPU multiplies by a rounded 1 / 448)
    assert sf[1, 3].item() == F.block_scale(x[3, 128:].nan_to_num(0).abs().max().cpu().numpy())
    assert v[4].isnan().all() and (sf[:, 4] == tiny).all()
    assert (v[5] == 448).all()
    w = torch.zeros(128, 128, device="cuda")
    w[3, 3] = torch.nan
    q, sf = ops.quantize_fp8_block_weight(w)
    assert sf.item() == np.float32(tiny) and q.view(torch.float8_e4m3fn).float().isnan().sum() == 1


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,k", [(1, 16), (5, 128), (33, 400), (64, 2048)])
def test_silu(rows, k, dtype):
    """The activation takes the approximate exponential and reciprocal: a few 2^-22 with 2^-24 |gate| of
    each value, so of the scale; a byte moves where a value lies that near a border."""
    from mosaicist_b200 import ops

    rng = np.random.default_rng([rows, k])
    x = T(rng.standard_normal((rows, 2 * k)).astype(np.float32) * 2).to(DT[dtype])
    q, sf = ops.quantize_fp8_block(x, silu=True)
    act = F.silu_mul(x.float().cpu().numpy())
    pad = np.pad(act, ((0, 0), (0, -k % 128))).reshape(rows, -1, 128)
    want = np.abs(pad).max(2).T / 448
    tol = 4 * 2.0 ** -22 + 12 * 2.0 ** -24          # |gate| < 12
    assert (np.abs(sf.cpu().numpy()[:, :rows] - want) <= tol * want + 2.0 ** -126).all()
    got = F.values(q.cpu().numpy())
    ratio = act / np.repeat(sf.cpu().numpy().T[:rows].astype(np.float64), 128, 1)[:, :k]
    # half a step of the value (2^-4 relative, 2^-10 below the normal range) and what the value may be off by
    assert (np.abs(got - np.clip(ratio, -448, 448)) <= np.maximum(np.abs(ratio) * 2.0 ** -4, 2.0 ** -10) * (1 + 1e-4) + 2 * tol * np.abs(ratio)).all()


@pytest.mark.parametrize("silu", [False, True])
def test_groups(silu):
    """Rows that no group owns stay as they are, and are not read; groups start anywhere, may be empty, in
    any order, and are cut where the rows end."""
    from mosaicist_b200 import ops

    rng = np.random.default_rng(2)
    total, k = 203, 272
    x = T(rng.standard_normal((total, k * (2 if silu else 1))).astype(np.float32)).bfloat16()
    offs, rows = [128, 3, 70, 40, 199, -4, 500, 60], [50, 20, 0, 17, 300, 3, 10, -5]
    live = np.zeros(total, bool)
    for o, r in zip(offs, rows):
        if 0 <= o < total and r > 0:
            live[o:o + r] = True
    want_q, want_sf = ops.quantize_fp8_block(x, silu=silu)
    x[torch.from_numpy(~live).cuda()] = torch.nan
    q = torch.full((total, k), 0x55, dtype=torch.uint8, device="cuda")
    sf = torch.full((3, 204), -7.0, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    got = ops.quantize_fp8_block(x, silu=silu, group_offsets=i32(offs), group_rows=i32(rows), out=(q, sf))
    assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == sf.data_ptr()
    lv = torch.from_numpy(live).cuda()
    assert torch.equal(q[lv], want_q[lv]) and (q[~lv] == 0x55).all()
    assert torch.equal(sf[:, :total][:, lv], want_sf[:, :total][:, lv]) and (sf[:, :total][:, ~lv] == -7).all()
    assert (sf[:, total:] == 0).all()
    import mosaicist_b200.torch_ops as O

    fresh = O.quantize_fp8_block(x, silu, i32(offs), i32(rows))
    assert torch.equal(fresh[0][lv], q[lv]) and (fresh[0][~lv] == 0).all() and (fresh[1][:, :total][:, ~lv] == 0).all()


# ---- products ------------------------------------------------------------------------------


def _operands(rng, rows, l, n, k, exact):
    """exact: small integers and scales that are powers of two, so that every sum is exact."""
    if exact:
        a = rng.integers(-4, 5, (rows, k)).astype(ml_dtypes.float8_e4m3fn).view(np.uint8)
        b = rng.integers(-3, 4, (l, n, k)).astype(ml_dtypes.float8_e4m3fn).view(np.uint8)
        sa = 2.0 ** rng.integers(-2, 3, (-(-k // 128), rows))
        sb = 2.0 ** rng.integers(-2, 3, (l, -(-n // 128), -(-k // 128)))
    else:
        a, sa = F.quantize_rows(_rows(rng, rows, k))
        parts = [F.quantize_weight((rng.standard_normal((n, k)) * 0.05).astype(np.float32)) for _ in range(l)]
        b, sb = np.stack([p[0] for p in parts]), np.stack([p[1] for p in parts])
    return a, sa.astype(np.float32), b, sb.astype(np.float32)


def _dev_sf(sa, poison=None):
    """The scales with their padded pitch."""
    pad = -sa.shape[1] % 4
    return T(np.pad(sa, ((0, 0), (0, pad)), constant_values=0 if poison is None else poison))


def _check(got, want, mags, k, dtype, exact):
    got = got.double().cpu().numpy()
    if exact:
        t = torch.from_numpy(want).to(DT[dtype]).double().numpy()
        assert np.array_equal(got, t)
        return
    # one rounding to the type; every addition in fp32 (128 in a block, the blocks, the scales' products) is
    # off by at most 2^-23 of the magnitudes' sum
    bound = HALF_STEP[dtype] * np.abs(want) + (128 + k // 128 + 4) * 2.0 ** -23 * mags
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / np.maximum(bound, 1e-300)).max())


DENSE = [(1, 8, 16), (1, 128, 128), (2, 256, 256), (3, 136, 144), (16, 512, 2048), (31, 264, 400), (32, 256, 128), (33, 256, 256),
         (65, 264, 1040), (96, 128, 384), (97, 384, 512), (129, 40, 272), (255, 256, 640), (256, 512, 512), (257, 256, 384),
         (288, 256, 256), (289, 520, 272), (300, 1000, 400), (545, 776, 1296), (777, 1048, 3088), (70, 512, 7168), (4, 1024, 7168)]


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("m,n,k", DENSE)
def test_dense(m, n, k, exact):
    from mosaicist_b200 import ops

    rng = np.random.default_rng([m, n, k])
    a, sa, b, sb = _operands(rng, m, 1, n, k, exact)
    want, mags = F.product(a, sa, b[0], sb[0])
    args = T(a), _dev_sf(sa), T(b[0]), T(sb[0])
    for dtype in DT:
        got = ops.gemm_fp8_block(*args, out_dtype=DT[dtype])
        assert got.dtype == DT[dtype]
        _check(got, want, mags, k, dtype, exact)
    again = ops.gemm_fp8_block(*args, out_dtype=torch.float32)
    few = ops.gemm_fp8_block(*args, out_dtype=torch.float32, max_ctas=6)
    assert torch.equal(again, ops.gemm_fp8_block(*args, out_dtype=torch.float32))     # the order of the sums is fixed
    _check(few, want, mags, k, "f32", exact)


@pytest.mark.parametrize("m,n,k,ctas", [(1792, 256, 272, 12), (1797, 256, 1040, 12), (1700, 256, 128, 12), (256, 264, 400, 16), (520, 1000, 272, 28),
                                        (100, 1304, 640, 0), (4101, 520, 272, 0)])
def test_last_round_in_quarter_tiles(m, n, k, ctas):
    """Grids whose last round of tiles would be nearly empty: those tiles are taken in quarters, some of which are empty."""
    from mosaicist_b200 import ops

    rng = np.random.default_rng([m, n, k])
    a, sa, b, sb = _operands(rng, m, 1, n, k, True)
    want = F.product(a, sa, b[0], sb[0])[0]
    out = torch.full((m + 9, n), 3.0, dtype=torch.float32, device="cuda")
    got = ops.gemm_fp8_block(T(a), _dev_sf(sa), T(b[0]), T(sb[0]), out=out[:m], max_ctas=ctas)
    _check(got, want, None, k, "f32", True)
    assert (out[m:] == 3).all()


@pytest.mark.parametrize("m,n,k", [(1, 264, 4112), (33, 1000, 4112), (64, 8, 6160), (200, 520, 7184), (300, 1304, 4112), (257, 256, 16400)])
def test_few_tiles_split_along_k(m, n, k):
    """Two and four shares of K, uneven ones too, of tiles of either kind."""
    from mosaicist_b200 import ops

    rng = np.random.default_rng([m, n, k])
    a, sa, b, sb = _operands(rng, m, 1, n, k, True)
    want = F.product(a, sa, b[0], sb[0])[0]
    out = torch.full((m + 9, n), 3.0, dtype=torch.float32, device="cuda")
    got = ops.gemm_fp8_block(T(a), _dev_sf(sa), T(b[0]), T(sb[0]), out=out[:m])
    _check(got, want, None, k, "f32", True)
    assert (out[m:] == 3).all()


def test_dense_writes_its_rows_only():
    from mosaicist_b200 import ops

    rng = np.random.default_rng(1)
    m, n, k = 67, 392, 272
    a, sa, b, sb = _operands(rng, m, 1, n, k, True)
    for dtype in DT:
        big = torch.full((m + 64, n), 7.0, dtype=DT[dtype], device="cuda")
        got = ops.gemm_fp8_block(T(a), _dev_sf(sa), T(b[0]), T(sb[0]), out=big[:m])
        assert got.data_ptr() == big.data_ptr() and (big[m:] == 7).all()
        _check(got, *F.product(a, sa, b[0], sb[0]), k, dtype, True)


GROUPED = [
    ([5], None), ([0, 1, 0, 33], None), ([256, 272, 288, 289], None), ([300, 0, 7, 520, 31, 64], None),
    ([1] * 70, None),                                     # more groups than a window of 32
    ([9, 40, 3, 130], [1, 67, 133, 202]),                 # groups that start anywhere
    ([40, 9, 70], [203, 130, 2]),                         # in any order
    ([30, 500, -3, 8, 8], [0, 100, 64, -8, 10 ** 6]),     # reaching beyond the rows, and beyond reason
]


@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("case", range(len(GROUPED)))
def test_grouped(case, scaled, exact):
    from mosaicist_b200 import ops

    rows, offs = GROUPED[case]
    if offs is None:
        offs, at = [], 0
        for r in rows:
            offs.append(at)
            at += -(-r // 128) * 128
        total = max(at, 128)
    else:
        total = 251
    l, n, k = len(rows), 264, 400
    rng = np.random.default_rng([case, scaled])
    a, sa, b, sb = _operands(rng, total, l, n, k, exact)
    rs = 2.0 ** rng.integers(-2, 3, total).astype(np.float32) if scaled else None
    want = np.full((total, n), -3.0)
    mags = np.zeros((total, n))
    live = np.zeros(total, bool)
    for g, (o, r) in enumerate(zip(offs, rows)):
        if 0 <= o < total and r > 0:
            e = min(o + r, total)
            y, m = F.product(a[o:e], sa[:, o:e], b[g], sb[g])
            f = rs[o:e, None] if scaled else 1.0
            want[o:e], mags[o:e] = y * f, m * f
            live[o:e] = True
    a[~live] = 0x7f                        # NaN where nobody owns a row
    sa[:, ~live] = np.nan
    if scaled:
        rs[~live] = np.nan
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for dtype in DT:
        out = torch.full((total, n), -3.0, dtype=DT[dtype], device="cuda")
        got = ops.ragged_grouped_gemm_fp8_block(T(a), _dev_sf(sa, np.nan), T(b), T(sb), i32(offs), i32(rows),
                                                None if rs is None else T(rs), out=out)
        assert got.data_ptr() == out.data_ptr()
        _check(got, want, mags, k, dtype, exact)


@pytest.mark.parametrize("k", [400, 2048, 4112])
@pytest.mark.parametrize("order", ["falling", "rising", "mixed"])
def test_one_pair_meets_tiles_of_every_width(order, k):
    """A single CTA pair works through tiles of one to nine units of 32 tokens: parts of the kernel sit some of them out,
    for fewer and for more K blocks than it has accumulators."""
    from mosaicist_b200 import ops

    rows = sorted([1, 20, 33, 64, 65, 96, 100, 130, 190, 200, 256, 280, 288, 290, 330])
    rows = rows[::-1] if order == "falling" else rows if order == "rising" else [rows[(7 * i) % 15] for i in range(15)]
    offs, at = [], 0
    for r in rows:
        offs.append(at)
        at += r
    l, n = len(rows), 136
    rng = np.random.default_rng(k)
    a, sa, b, sb = _operands(rng, at, l, n, k, True)
    want = np.concatenate([F.product(a[o:o + r], sa[:, o:o + r], b[g], sb[g])[0] for g, (o, r) in enumerate(zip(offs, rows))])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for ctas in (2, 4, 0):
        got = ops.ragged_grouped_gemm_fp8_block(T(a), _dev_sf(sa), T(b), T(sb), i32(offs), i32(rows), out_dtype=torch.float32, max_ctas=ctas)
        _check(got, want, None, k, "f32", True)


def test_views_streams_graphs_and_float8():
    """Operands as float8 tensors and as slices at an offset; another stream; a captured call replayed on new data."""
    from mosaicist_b200 import ops

    rng = np.random.default_rng(9)
    m, n, k = 48, 256, 512
    a, sa, b, sb = _operands(rng, m, 1, n, k, True)
    want = F.product(a, sa, b[0], sb[0])
    da, ds, db, dsb = T(a), _dev_sf(sa), T(b[0]), T(sb[0])
    e4 = torch.float8_e4m3fn
    _check(ops.gemm_fp8_block(da.view(e4), ds, db.view(e4), dsb), *want, k, "bf16", True)
    wide = torch.zeros(m + 3, k, dtype=torch.uint8, device="cuda")
    wide[3:] = da
    _check(ops.gemm_fp8_block(wide[3:], ds, db, dsb), *want, k, "bf16", True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.gemm_fp8_block(da, ds, db, dsb)
    s.synchronize()
    _check(got, *want, k, "bf16", True)
    x = torch.randn(m, k, device="cuda").bfloat16()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, sf = ops.quantize_fp8_block(x)
        held = ops.gemm_fp8_block(q, sf, db, dsb)
    x.copy_(torch.randn(m, k, device="cuda"))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, ops.gemm_fp8_block(*ops.quantize_fp8_block(x), db, dsb))
    assert ops.gemm_fp8_block(da[:0], ds[:, :0], db, dsb).shape == (0, n)
    assert ops.quantize_fp8_block(x[:0])[1].shape == (k // 128, 0)


def test_torch_operators():
    import mosaicist_b200.torch_ops as O
    from mosaicist_b200 import ops

    x, w = torch.randn(40, 272, device="cuda").bfloat16(), torch.randn(2, 136, 272, device="cuda")
    q, sf = O.quantize_fp8_block(x, False, None, None)
    wq, wsf = O.quantize_fp8_block_weight(w)
    want = ops.gemm_fp8_block(q, sf, wq[1], wsf[1], out_dtype=torch.float32)
    assert torch.equal(O.gemm_fp8_block(q, sf, wq[1], wsf[1], torch.float32), want)
    offs, rows = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 20], [10, 15]))
    y = O.grouped_gemm_fp8_block_ragged(q, sf, wq, wsf, offs, rows, None, torch.float16)
    assert torch.equal(y[20:35], want[20:35].half()) and (y[10:20] == 0).all() and (y[35:] == 0).all()


@pytest.mark.parametrize("rows", [[64, 64, 64], [256, 256], [63, 65, 62, 64], [255, 257, 256, 1], [512, 64]])
def test_whole_tiles_at_odd_rows(rows):
    """Groups of whole tiles that start on any row, a row between them that nobody owns."""
    from mosaicist_b200 import ops

    n, k = 392, 528
    offs, at = [], 3
    for r in rows:
        offs.append(at)
        at += r + 1
    rng = np.random.default_rng(rows)
    a, sa, b, sb = _operands(rng, at, len(rows), n, k, True)
    want = np.full((at, n), -3.0)
    for g, (o, r) in enumerate(zip(offs, rows)):
        want[o:o + r] = F.product(a[o:o + r], sa[:, o:o + r], b[g], sb[g])[0]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for dtype in DT:
        out = torch.full((at, n), -3.0, dtype=DT[dtype], device="cuda")
        ops.ragged_grouped_gemm_fp8_block(T(a), _dev_sf(sa), T(b), T(sb), i32(offs), i32(rows), out=out)
        _check(out, want, None, k, dtype, True)


def test_empty_batches_check_their_sizes():
    from mosaicist_b200 import _lib, ops

    u8, f32 = dict(dtype=torch.uint8, device="cuda"), dict(device="cuda")
    assert ops.quantize_fp8_block(torch.empty(0, 64, **f32))[0].shape == (0, 64)
    assert ops.gemm_fp8_block(torch.empty(0, 64, **u8), torch.empty(1, 0, **f32), torch.empty(16, 64, **u8), torch.empty(1, 1, **f32)).shape == (0, 16)
    with pytest.raises(_lib.MscError, match="k=100"):
        ops.quantize_fp8_block(torch.empty(0, 100, **f32))
    with pytest.raises(_lib.MscError, match="n=20"):
        ops.gemm_fp8_block(torch.empty(0, 64, **u8), torch.empty(1, 0, **f32), torch.empty(20, 64, **u8), torch.empty(1, 1, **f32))
