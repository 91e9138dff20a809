"""QuantizeBlocks, MatMulBlocks and TokenLogProbs against their definitions in 64 bits (tests/scoring_reference.py)."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")  # before the library, which then shares torch's HIP runtime

import scoring_reference as R
from scoring_reference import E4M3, E5M2

pytestmark = pytest.mark.gpu


def dev(hip, a, element_type=None, offset=0):
    """a on the device; offset: elements past a 256-byte boundary."""
    a = np.ascontiguousarray(a).reshape(np.shape(a))
    if not offset:
        return hip.DeviceTensor.from_numpy(a, element_type)
    flat = np.concatenate([np.zeros(offset, a.dtype), a.reshape(-1)])
    t = hip.DeviceTensor.from_numpy(flat, element_type)
    at = t.h.data + offset * a.itemsize
    return hip.DeviceTensor.wrap(at, a.shape, a.dtype if element_type is None else element_type, a.nbytes, keepalive=t)


def ok(r):
    assert r.Status.name == "Success", r.Message
    return [t.to_numpy() for t in r.Outputs]


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def near(got, want, err):
    want, err = np.asarray(want), np.broadcast_to(err, np.shape(want))
    assert got.shape == want.shape
    fin = np.isfinite(want)
    assert same(got[~fin].astype(np.float64), want[~fin])
    off = np.abs(got[fin].astype(np.float64) - want[fin])
    assert (off <= err[fin]).all(), (float(off.max()), float((off / err[fin]).max()))


# ---- QuantizeBlocks -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 127), (5, 129), (128, 128), (129, 257), (2, 3, 384), (3, 130, 36),
                                   (200, 1000), (1, 8192), (2, 2, 131, 260)])
def test_quantize(hip, shape, block_rows, fmt):
    rng = np.random.default_rng([sum(shape), fmt, block_rows])
    x = (rng.standard_normal(shape) * np.exp(2 * rng.standard_normal(shape[-1]))).astype(np.float32)
    q, s = ok(hip.HipExecutionProvider.QuantizeBlocks(dev(hip, x), to=fmt, block_rows=block_rows))
    val, scale = R.quantize(x, fmt, block_rows)
    assert s.dtype == np.float32 and s.shape == scale.shape and np.array_equal(s, scale)
    assert q.shape == x.shape and same(R.decode(q, fmt), val)
    assert same(np.signbit(R.decode(q, fmt)), np.signbit(x))


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_quantize_vector_and_unaligned_storage(hip, fmt):
    x = np.random.default_rng(fmt).standard_normal((70, 256)).astype(np.float32)
    val, scale = R.quantize(x, fmt, 1)
    for offset in (1, 2, 3):
        q, s = ok(hip.HipExecutionProvider.QuantizeBlocks(dev(hip, x, offset=offset), to=fmt))
        assert np.array_equal(s, scale) and same(R.decode(q, fmt), val)
    val, scale = R.quantize(x[0], fmt, 1)
    q, s = ok(hip.HipExecutionProvider.QuantizeBlocks(dev(hip, x[0]), to=fmt))  # a vector
    assert s.shape == (2,) and np.array_equal(s, scale) and same(R.decode(q, fmt), val)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("power", [-140, -127, -100, -63, -20, 0, 60, 110])
def test_quantize_every_middle_and_its_neighbours(hip, fmt, power):
    """Each code, the middle to the next one and the floats on both sides of the middle, in blocks whose scale is a
    power of two (quotients exact) and one that is not (quotients of every kind), at both ends of float's range."""
    grid = R.VALUES[fmt][:128]
    grid = grid[np.isfinite(grid)]
    mid = ((grid[1:] + grid[:-1]) / 2).astype(np.float32)
    v = np.concatenate([grid.astype(np.float32), mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e9))])
    v = np.concatenate([v, -v])
    v = np.concatenate([v, np.zeros(-len(v) % 127, np.float32)]).reshape(-1, 127)
    for f in (1.0, 1.37):
        top = np.float32(R.MAX[fmt])
        with np.errstate(under="ignore"):
            x = (np.concatenate([np.full((len(v), 1), top), v], 1).astype(np.float64) * f * 2.0 ** power).astype(np.float32)
        q, s = ok(hip.HipExecutionProvider.QuantizeBlocks(dev(hip, x), to=fmt))
        val, scale = R.quantize(x, fmt, 1)
        assert np.array_equal(s, scale) and same(R.decode(q, fmt), val)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(hip, fmt, block_rows):
    inf, nan, big = np.inf, np.nan, np.finfo(np.float32).max
    x = np.zeros((6, 256), np.float32)
    x[1, :4] = [inf, -inf, nan, 3.0]
    x[2, :3] = [nan, inf, 0.0]           # nothing finite but zeros
    x[3, :3] = [big, -big, 1e-30]
    x[4, :3] = [2.0 ** -149, -(2.0 ** -149), 2.0 ** -130]
    x[5, 128:131] = [-0.0, 1.0, -inf]
    for rows in (x, x[2:3], x[4:5]):
        q, s = ok(hip.HipExecutionProvider.QuantizeBlocks(dev(hip, rows), to=fmt, block_rows=block_rows))
        val, scale = R.quantize(rows, fmt, block_rows)
        assert np.array_equal(s, scale) and same(R.decode(q, fmt), val)


def test_quantize_empty(hip):
    for shape, sshape in (((0, 128), (0, 1)), ((3, 0), (3, 0)), ((0,), (0,))):
        q, s = ok(hip.HipExecutionProvider.QuantizeBlocks(dev(hip, np.zeros(shape, np.float32))))
        assert q.shape == shape and s.shape == sshape


# ---- MatMulBlocks ---------------------------------------------------------------------------------------------
def operand(rng, rows, k, fmt, by_row, spread=1.0):
    c = rng.integers(0, 256, (rows, k)).astype(np.uint8)
    c = np.where(np.isfinite(R.decode(c, fmt)), c, 0x30).astype(np.uint8)
    s = np.exp(spread * rng.standard_normal((rows if by_row else R.blocks(rows), R.blocks(k)))).astype(np.float32)
    return c, s


def product(hip, a, sa, fa, b, sb, fb, bias=None, offset=0):
    HIP = hip.HipExecutionProvider
    y, = ok(HIP.MatMulBlocks(dev(hip, a, fa, offset), dev(hip, sa), dev(hip, b, fb, offset), dev(hip, sb),
                             bias=None if bias is None else dev(hip, bias)))
    return y


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 384, 384), (2, 129, 33), (7, 127, 130), (31, 512, 96), (33, 640, 257), (64, 256, 64),
          (65, 2048, 100), (1, 4096, 515), (16, 16, 16), (100, 1111, 77), (129, 768, 384), (128, 144, 1000), (257, 400, 300),
          (300, 384, 513), (1000, 272, 129), (512, 1536, 640), (1, 20000, 5),
          (3, 256, 8300), (3, 77, 8300), (200, 333, 1500), (500, 384, 1030), (500, 301, 1030), (1040, 400, 1030), (1088, 256, 1088),
          (2000, 272, 2100), (2049, 128, 2051), (2000, 131, 2100), (2048, 640, 2048),
          (4100, 128, 2060), (4100, 144, 2063)]  # results past the caches


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("by_row", [False, True])
def test_matmul(hip, m, k, n, by_row):
    rng = np.random.default_rng([m, k, n, by_row])
    fa, fb = [(E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)][(m + k + n) % 4]
    (a, sa), (b, sb) = operand(rng, m, k, fa, True), operand(rng, n, k, fb, by_row)
    bias = rng.standard_normal(n).astype(np.float32) if (m + n) % 2 else None
    y = product(hip, a, sa, fa, b, sb, fb, bias)
    near(y, *R.matmul(R.decode(a, fa), sa, R.decode(b, fb), sb, bias))


@pytest.mark.parametrize("fa", [E4M3, E5M2])
@pytest.mark.parametrize("fb", [E4M3, E5M2])
@pytest.mark.parametrize("m,k,n", [(1, 300, 70), (40, 256, 130), (260, 384, 200), (500, 144, 1030), (1040, 144, 1030),
                                   (2000, 144, 2100)])
def test_matmul_every_pair_of_types_and_alignment(hip, fa, fb, m, k, n):
    rng = np.random.default_rng([fa, fb, m])
    (a, sa), (b, sb) = operand(rng, m, k, fa, True), operand(rng, n, k, fb, False)
    want = R.matmul(R.decode(a, fa), sa, R.decode(b, fb), sb)
    for offset in (0, 1, 8):
        near(product(hip, a, sa, fa, b, sb, fb, offset=offset), *want)


@pytest.mark.parametrize("m,k,n", [(1, 1024, 128), (5, 130, 260), (70, 384, 33), (256, 640, 384), (513, 128, 1025),
                                   (1040, 640, 1030), (2000, 400, 2100)])
@pytest.mark.parametrize("by_row", [False, True])
def test_matmul_is_exact_where_float_is(hip, m, k, n, by_row):
    """Small whole values with scales that are powers of two: every sum is a float, whatever its order."""
    rng = np.random.default_rng([m, k, n])
    small = np.flatnonzero(np.isin(R.VALUES[E4M3], [-4, -3, -2, -1, 0, 1, 2, 3, 4])).astype(np.uint8)
    a, b = rng.choice(small, (m, k)), rng.choice(small, (n, k))
    sa = (2.0 ** rng.integers(-2, 3, (m, R.blocks(k)))).astype(np.float32)
    sb = (2.0 ** rng.integers(-2, 3, (n if by_row else R.blocks(n), R.blocks(k)))).astype(np.float32)
    bias = rng.integers(-8, 9, n).astype(np.float32)
    want, _ = R.matmul(R.decode(a, E4M3), sa, R.decode(b, E4M3), sb, bias)
    assert np.array_equal(product(hip, a, sa, E4M3, b, sb, E4M3, bias), want)


@pytest.mark.parametrize("m,n", [(3, 40), (200, 300), (520, 1030), (1040, 1030), (2000, 2100)])
def test_matmul_special_values(hip, m, n):
    """NaN and infinite codes reach the rows and columns that hold them and no others; scales of zero count."""
    k = 272
    rng = np.random.default_rng(m)
    (a, sa), (b, sb) = operand(rng, m, k, E4M3, True), operand(rng, n, k, E5M2, True)
    a[1, k - 1] = 0x7f                       # NaN, last of the row: its neighbours in memory are row 2's
    b[2, 3], b[n - 1, k - 1] = 0x7c, 0xfe    # inf; NaN
    a[:, 3] = 0x38                           # 1.0 against the infinity
    sa[0, 1], sb[5, :] = 0.0, 0.0
    va, vb = R.decode(a, E4M3), R.decode(b, E5M2)
    with np.errstate(invalid="ignore"):
        want, err = R.matmul(np.nan_to_num(va, nan=0.0), sa, np.nan_to_num(vb, nan=0.0, posinf=0.0), sb)
    want[:, 2] = np.inf
    want[1, :] = np.nan
    want[:, n - 1] = np.nan
    near(product(hip, a, sa, E4M3, b, sb, E5M2), want, err)


def test_matmul_leading_axes_and_empty(hip):
    HIP = hip.HipExecutionProvider
    rng = np.random.default_rng(5)
    (a, sa), (b, sb) = operand(rng, 6, 200, E4M3, True), operand(rng, 50, 200, E4M3, False)
    want, err = R.matmul(R.decode(a, E4M3), sa, R.decode(b, E4M3), sb)
    db, dsb = dev(hip, b, E4M3), dev(hip, sb)
    y, = ok(HIP.MatMulBlocks(dev(hip, a.reshape(2, 1, 3, 200), E4M3), dev(hip, sa.reshape(2, 1, 3, 2)), db, dsb))
    near(y, want.reshape(2, 1, 3, 50), err.reshape(2, 1, 3, 50))
    y, = ok(HIP.MatMulBlocks(dev(hip, a[2], E4M3), dev(hip, sa[2]), db, dsb))  # one token's vector
    near(y, want[2], err[2])
    y, = ok(HIP.MatMulBlocks(dev(hip, a[:0], E4M3), dev(hip, sa[:0]), db, dsb))
    assert y.shape == (0, 50)
    bias = rng.standard_normal(4).astype(np.float32)
    e = np.zeros((3, 0), np.uint8), np.zeros((3, 0), np.float32), np.zeros((4, 0), np.uint8), np.zeros((1, 0), np.float32)
    args = [dev(hip, e[0], E4M3), dev(hip, e[1]), dev(hip, e[2], E4M3), dev(hip, e[3])]
    assert np.array_equal(ok(HIP.MatMulBlocks(*args))[0], np.zeros((3, 4), np.float32))
    assert np.array_equal(ok(HIP.MatMulBlocks(*args, bias=dev(hip, bias)))[0], np.broadcast_to(bias, (3, 4)))


def test_matmul_writes_its_own_rows_only(hip):
    """The storage behind the last row, and the rows of a larger buffer, stay as they were."""
    rng = np.random.default_rng(9)
    for m, k, n in ((5, 384, 130), (130, 256, 260), (500, 384, 1031), (1033, 144, 1030), (2000, 272, 2102)):
        (a, sa), (b, sb) = operand(rng, m, k, E4M3, True), operand(rng, n, k, E4M3, False)
        big = dev(hip, np.full((m + 2, n), 7.0, np.float32))
        out = hip.DeviceTensor.wrap(big.h.data + 4 * n, (m, n), np.float32, 4 * m * n, keepalive=big)
        y, = ok(hip.HipExecutionProvider.MatMulBlocks(dev(hip, a, E4M3), dev(hip, sa), dev(hip, b, E4M3), dev(hip, sb), out=out))
        near(y, *R.matmul(R.decode(a, E4M3), sa, R.decode(b, E4M3), sb))
        whole = big.to_numpy()
        assert (whole[0] == 7).all() and (whole[-1] == 7).all()


# ---- TokenLogProbs --------------------------------------------------------------------------------------------
def check_logprobs(hip, x, ids=None, top=0, entropy=True, offset=0, ids_type=np.int64):
    x = np.asarray(x, np.float32)
    r = hip.HipExecutionProvider.TokenLogProbs(dev(hip, x, offset=offset), None if ids is None else dev(hip, np.asarray(ids, ids_type)),
                                               top=top, entropy=entropy)
    got = ok(r)
    want = R.logprobs(x.reshape(-1, x.shape[-1]), None if ids is None else np.reshape(ids, -1), top)
    lead = x.shape[:-1]
    if ids is not None:
        near(got.pop(0), want["lp"].reshape(lead), want["lp_err"].reshape(lead))
    if entropy:
        near(got.pop(0), want["h"].reshape(lead), want["h_err"].reshape(lead))
    if top:
        assert np.array_equal(got.pop(0), want["top_ids"].reshape(lead + (top,)))
        near(got.pop(0), want["top_lp"].reshape(lead + (top,)), want["top_lp_err"].reshape(lead + (top,)))
    assert not got


@pytest.mark.parametrize("t,v", [(1, 1), (1, 2), (3, 5), (2, 63), (5, 64), (4, 257), (7, 1001), (3, 4095), (9, 8193), (2, 30522),
                                 (300, 515), (1, 131072), (1, 200003), (65, 20001), (1100, 3001)])
@pytest.mark.parametrize("top", [0, 1, 5, 64])
def test_logprobs(hip, t, v, top):
    rng = np.random.default_rng([t, v, top])
    x = 3 * rng.standard_normal((t, v))
    ids = rng.integers(-2, v + 1, t)
    check_logprobs(hip, x, ids, min(top, v), ids_type=np.int32 if t % 2 else np.int64)


@pytest.mark.parametrize("v", [9, 1023, 5001, 70001])
def test_logprobs_rows_at_any_offset_and_shape(hip, v):
    rng = np.random.default_rng(v)
    x = rng.standard_normal((2, 3, v)) * 4
    for offset in (0, 1, 2, 3):
        check_logprobs(hip, x, rng.integers(0, v, (2, 3)), 3, offset=offset)
    check_logprobs(hip, x[0, 0], np.int64(4), 2)   # one row without leading axes
    check_logprobs(hip, x, None, 2, entropy=False)
    check_logprobs(hip, x, None, 0)
    check_logprobs(hip, x, rng.integers(0, v, (2, 3)), 0, entropy=False)


@pytest.mark.parametrize("v", [40, 700, 9000, 131072])
def test_logprobs_masks_ties_and_special_values(hip, v):
    rng = np.random.default_rng(v)
    low = np.finfo(np.float32).min
    x = rng.standard_normal((18, v)).astype(np.float32)
    x[0] = 1.25                                   # uniform
    x[1] = -np.inf                                # a mask that leaves nothing
    x[2] = low                                    # all the lowest value: uniform
    x[3, rng.permutation(v)[:v // 2]] = low
    x[4] = -np.inf; x[4, v // 2] = 3.0            # one token left: certain
    x[5] = -np.inf; x[5, [1, v - 1]] = -2.0       # two left, fewer than asked for
    x[6, v - 1] = np.nan
    x[7, 0] = np.inf
    x[8] = np.round(x[8])                         # many equal logits
    x[9] = np.where(rng.random(v) < .5, 0.0, -0.0)
    x[10] = np.sort(x[10])
    x[11] = np.sort(x[11])[::-1]
    x[12] = -60.0; x[12, 3] = 0.0                 # all but certain
    x[13] = np.finfo(np.float32).max; x[13, 7] = low
    x[14] = np.nan
    x[15, 1:] = np.nan
    x[16] = np.arange(v) % 7
    x[17] *= 1e30
    ids = rng.integers(0, v, 18)
    ids[12], ids[4] = 3, v // 2
    for top in (0, 1, 20, 40):
        check_logprobs(hip, x, ids, top)


def test_logprobs_keep_the_digits_of_near_certainty(hip):
    """log p of the likely token is about -exp(-17): relative to itself it still has float's digits."""
    for v in (16, 3000, 100000):
        x = np.full((1, v), -40.0, np.float32)
        x[0, 5], x[0, 9] = 0.0, -17.0
        lp, h = ok(hip.HipExecutionProvider.TokenLogProbs(dev(hip, x), dev(hip, np.array([5])), entropy=True))
        e = np.exp(np.array([-17.0] + [-40.0] * (v - 2)))
        want, wh = -np.log1p(e.sum()), np.log1p(e.sum()) + (e * -np.log(e)).sum() / (1 + e.sum())
        assert abs(lp[0] / want - 1) < 64 * R.U and abs(h[0] / wh - 1) < 64 * R.U


def test_logprobs_sorted_rows_overflow_the_candidate_buffer(hip):
    """Rows whose large logits all fall to few threads: the candidates exceed what is ranked at once."""
    v = 1024 * 90
    i = np.arange(v)
    x = np.zeros((1100, v), np.float32)   # more rows than are split
    x[:] = -(i // 1024).astype(np.float32) - 1000.0 * ((i // 4) % 256 >= 64)
    x[1::2] += (i % 4096) * 1e-3
    got = ok(hip.HipExecutionProvider.TokenLogProbs(dev(hip, x), top=64))
    for r in (0, 1, 1098, 1099):
        want = R.logprobs(x[r:r + 1], None, 64)
        assert np.array_equal(got[0][r], want["top_ids"][0])
        near(got[1][r], want["top_lp"][0], want["top_lp_err"][0])


def test_logprobs_are_the_same_from_run_to_run(hip):
    rng = np.random.default_rng(3)
    for t, v in ((1, 131072), (600, 5000)):
        x, ids = dev(hip, rng.standard_normal((t, v)).astype(np.float32)), dev(hip, rng.integers(0, v, t))
        first = ok(hip.HipExecutionProvider.TokenLogProbs(x, ids, top=10, entropy=True))
        for _ in range(3):
            again = ok(hip.HipExecutionProvider.TokenLogProbs(x, ids, top=10, entropy=True))
            assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_logprobs_empty(hip):
    lp, h, i, t = ok(hip.HipExecutionProvider.TokenLogProbs(dev(hip, np.zeros((0, 9), np.float32)), dev(hip, np.zeros(0, np.int64)),
                                                            top=2, entropy=True))
    assert lp.shape == h.shape == (0,) and i.shape == t.shape == (0, 2)


# ---- together ---------------------------------------------------------------------------------------------------
def head(hip, x, w, sw, bias, ids, outs):
    HIP = hip.HipExecutionProvider
    for r in (HIP.QuantizeBlocks(x, out=outs[:2]), HIP.MatMulBlocks(outs[0], outs[1], w, sw, bias=bias, out=outs[2]),
              HIP.TokenLogProbs(outs[2], ids, top=4, entropy=True, out=outs[3:])):
        assert r.Status.name == "Success", r.Message


@pytest.mark.parametrize("t,k,v", [(1, 384, 30522), (13, 768, 5003), (300, 128, 2000)])
def test_scoring_head(hip, t, k, v):
    """Hidden states to scores: each operator's outputs against its definition on the inputs it got."""
    rng = np.random.default_rng([t, k, v])
    x = rng.standard_normal((t, k)).astype(np.float32)
    wf = (rng.standard_normal((v, k)) / np.sqrt(k) * 3).astype(np.float32)
    bias = rng.standard_normal(v).astype(np.float32)
    ids = rng.integers(-1, v, t)
    E = hip.DeviceTensor.empty
    w, sw = hip.HipExecutionProvider.QuantizeBlocks(dev(hip, wf), block_rows=128).Outputs
    outs = (E((t, k), E4M3), E((t, R.blocks(k)), np.float32), E((t, v), np.float32), E((t,), np.float32), E((t,), np.float32),
            E((t, 4), np.int64), E((t, 4), np.float32))
    head(hip, dev(hip, x), w, sw, dev(hip, bias), dev(hip, ids), outs)
    q, s, y, lp, h, top, top_lp = (o.to_numpy() for o in outs)
    val, scale = R.quantize(x, E4M3, 1)
    assert np.array_equal(s, scale) and same(R.decode(q, E4M3), val)
    near(y, *R.matmul(val, s, R.decode(w.to_numpy(), E4M3), sw.to_numpy(), bias))
    want = R.logprobs(y, ids, 4)
    near(lp, want["lp"], want["lp_err"])
    near(h, want["h"], want["h_err"])
    assert np.array_equal(top, want["top_ids"])
    near(top_lp, want["top_lp"], want["top_lp_err"])
    # the 8-bit head says what the Float head says, within what three mantissa bits keep
    full = R.logprobs((x.astype(np.float64) @ wf.T.astype(np.float64) + bias).astype(np.float32), ids, 0)
    assert np.abs(full["lp"] - lp).max() < 1.0


def test_scoring_head_captured_and_replayed(hip):
    """The three calls recorded once into a graph, on a stream of the caller's, and replayed on new hidden states
    with eager calls of the same operators between."""
    rng = np.random.default_rng(1)
    t, k, v = 2, 256, 40000   # rows split over workgroups: partial results live in the graph's own memory
    HIP = hip.HipExecutionProvider
    f32 = torch.float32
    x = torch.empty((t, k), device="cuda", dtype=f32)
    wrap = hip.DeviceTensor.wrap_torch
    w, sw = HIP.QuantizeBlocks(dev(hip, (rng.standard_normal((v, k)) / 5).astype(np.float32)), block_rows=128).Outputs
    bias, ids = dev(hip, rng.standard_normal(v).astype(np.float32)), dev(hip, rng.integers(0, v, t))

    def buffers():
        return [torch.empty((t, k), device="cuda", dtype=torch.float8_e4m3fn), torch.empty((t, 2), device="cuda", dtype=f32),
                torch.empty((t, v), device="cuda", dtype=f32), torch.empty(t, device="cuda", dtype=f32),
                torch.empty(t, device="cuda", dtype=f32), torch.empty((t, 4), device="cuda", dtype=torch.int64),
                torch.empty((t, 4), device="cuda", dtype=f32)]

    rec, eager = buffers(), buffers()
    wrec, weager = [wrap(b) for b in rec], [wrap(b) for b in eager]
    x.copy_(torch.from_numpy(rng.standard_normal((t, k)).astype(np.float32)))
    head(hip, wrap(x), w, sw, bias, ids, weager)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs = []
    try:
        for _ in range(2):  # two graphs of the same calls
            graph = torch.cuda.CUDAGraph()
            hip.set_stream(stream.cuda_stream)
            with torch.cuda.graph(graph, stream=stream):
                head(hip, wrap(x), w, sw, bias, ids, wrec)
            hip.set_stream(None)
            graphs.append(graph)
    finally:
        hip.set_stream(None)
    for i in range(6):
        x.copy_(torch.from_numpy((i + 1) * rng.standard_normal((t, k)).astype(np.float32)))
        torch.cuda.synchronize()
        for b in rec:
            b.zero_()
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        head(hip, wrap(x), w, sw, bias, ids, weager)
        hip.synchronize()
        for a, b in zip(rec, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_product_of_odd_rows_captured_and_replayed(hip):
    """A product that copies its rows first: the copy lives in the graph's own memory."""
    rng = np.random.default_rng(2)
    m, k, n = 1100, 385, 1100
    (a, sa), (b, sb) = operand(rng, m, k, E4M3, True), operand(rng, n, k, E5M2, False)
    HIP, wrap = hip.HipExecutionProvider, hip.DeviceTensor.wrap_torch
    ta = torch.from_numpy(a).cuda().view(torch.float8_e4m3fn)
    args = [wrap(ta), dev(hip, sa), dev(hip, b, E5M2), dev(hip, sb)]
    y = torch.empty((m, n), device="cuda")
    wy = wrap(y)
    assert HIP.MatMulBlocks(*args, out=wy).Code == 0
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        hip.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            assert HIP.MatMulBlocks(*args, out=wy).Code == 0
    finally:
        hip.set_stream(None)
    for i in range(4):
        c = np.roll(a, i, 0)
        ta.view(torch.uint8).copy_(torch.from_numpy(c))
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = y.cpu().numpy()
        eager, = ok(HIP.MatMulBlocks(*args))
        assert np.array_equal(replayed, eager)
        near(eager, *R.matmul(R.decode(c, E4M3), sa, R.decode(b, E5M2), sb))


def test_products_on_another_stream_follow_its_work(hip):
    """set_stream: operands written on that stream just before, outputs read on it just after."""
    rng = np.random.default_rng(4)
    (a, sa), (b, sb) = operand(rng, 70, 512, E4M3, True), operand(rng, 300, 512, E4M3, False)
    want, err = R.matmul(R.decode(a, E4M3), sa, R.decode(b, E4M3), sb)
    src, ta = torch.from_numpy(a).cuda(), torch.zeros((70, 512), device="cuda", dtype=torch.uint8)
    y = torch.empty((70, 300), device="cuda")
    args = [hip.DeviceTensor.wrap_torch(ta.view(torch.float8_e4m3fn)), dev(hip, sa), dev(hip, b, E4M3), dev(hip, sb)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    try:
        hip.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            ta.copy_(src)
            assert hip.HipExecutionProvider.MatMulBlocks(*args, out=hip.DeviceTensor.wrap_torch(y)).Code == 0
            got = y.cpu().numpy()
    finally:
        hip.set_stream(None)
    near(got, want, err)


# ---- refusals ---------------------------------------------------------------------------------------------------
def refused(r, code, part=""):
    assert r.Status.name == "Failure" and r.Code == code and part in r.Message, (r.Code, r.Message)


def test_refusals(hip):
    from onnx_amd import _lib as L
    HIP, E = hip.HipExecutionProvider, hip.DeviceTensor.empty
    f32 = np.float32
    x = E((4, 256), f32)
    Q = HIP.QuantizeBlocks
    refused(Q(None), L.ERR_MISSING_INPUT, "X")
    refused(Q(E((4, 256), np.float64)), L.ERR_INPUT_TYPE_NOT_SUPPORTED, "Double")
    refused(Q(x, to=1), L.ERR_ATTRIBUTE_NOT_SUPPORTED, "to")
    refused(Q(x, to=18), L.ERR_ATTRIBUTE_NOT_SUPPORTED, "to")
    refused(Q(x, block_rows=64), L.ERR_ATTRIBUTE_NOT_SUPPORTED, "block_rows")
    refused(Q(E((), f32)), L.ERR_WRONG_INPUT_SHAPE)
    refused(Q(E((256,), f32), block_rows=128), L.ERR_WRONG_INPUT_SHAPE)
    refused(Q(x, out=(E((4, 255), E4M3), E((4, 2), f32))), L.ERR_BUFFER_TOO_SMALL)
    refused(Q(x, out=(E((4, 256), E4M3), E((4, 1), f32))), L.ERR_BUFFER_TOO_SMALL)
    inside = hip.DeviceTensor.wrap(x.h.data, (4, 256), E4M3, 1024, keepalive=x)
    refused(Q(x, out=(inside, E((4, 2), f32))), L.ERR_INVALID_ARGUMENT, "shares storage")
    odd = hip.DeviceTensor.wrap(x.h.data + 2, (4, 200), f32, 3200, keepalive=x)
    refused(Q(odd), L.ERR_INVALID_ARGUMENT, "aligned")
    with pytest.raises(ValueError):
        Q(x, out=(inside,))

    M = HIP.MatMulBlocks
    a, sa, b, sb = E((4, 256), E4M3), E((4, 2), f32), E((300, 256), E5M2), E((3, 2), f32)
    assert M(a, sa, b, sb).Code == 0
    for i, name in enumerate(("A", "a_scale", "B", "b_scale")):
        args = [a, sa, b, sb]
        args[i] = None
        refused(M(*args), L.ERR_MISSING_INPUT, name)
        args[i] = E([a, sa, b, sb][i].shape, np.int32)
        refused(M(*args), L.ERR_INPUT_TYPE_NOT_SUPPORTED, name)
    refused(M(a, sa, b, sb, bias=E((300,), np.float64)), L.ERR_INPUT_TYPE_NOT_SUPPORTED, "bias")
    refused(M(E((), E4M3), sa, b, sb), L.ERR_WRONG_INPUT_SHAPE, "A")
    refused(M(a, sa, E((1, 300, 256), E4M3), sb), L.ERR_WRONG_INPUT_SHAPE, "B")
    refused(M(a, sa, E((300, 255), E4M3), sb), L.ERR_INVALID_ARGUMENT, "columns")
    refused(M(a, E((4, 3), f32), b, sb), L.ERR_WRONG_INPUT_SHAPE, "a_scale")
    refused(M(a, E((8,), f32), b, sb), L.ERR_WRONG_INPUT_SHAPE, "a_scale")
    refused(M(a, sa, b, E((2, 2), f32)), L.ERR_WRONG_INPUT_SHAPE, "b_scale")
    refused(M(a, sa, b, E((2, 3), f32)), L.ERR_WRONG_INPUT_SHAPE, "b_scale")
    refused(M(a, sa, b, sb, bias=E((299,), f32)), L.ERR_WRONG_INPUT_SHAPE, "bias")
    refused(M(a, sa, b, sb, out=E((4, 299), f32)), L.ERR_BUFFER_TOO_SMALL)
    refused(M(E((1, 1 << 23), E4M3), E((1, 1 << 16), f32), E((1, 1 << 23), E4M3), E((1, 1 << 16), f32)), L.ERR_NOT_SUPPORTED, "2^23")
    many = E((131072, 1), E4M3), E((131072, 1), f32), E((65568, 1), E4M3), E((513, 1), f32)
    refused(M(*many), L.ERR_NOT_SUPPORTED, "2^23")
    big = E((4, 300), f32)
    inside = hip.DeviceTensor.wrap(big.h.data + 128, (4, 256), E4M3, 1024, keepalive=big)
    refused(M(inside, sa, b, sb, out=big), L.ERR_INVALID_ARGUMENT, "shares storage")

    T = HIP.TokenLogProbs
    y, ids = E((4, 50), f32), E((4,), np.int32)
    refused(T(None, entropy=True), L.ERR_MISSING_INPUT, "logits")
    refused(T(E((4, 50), np.float64), ids), L.ERR_INPUT_TYPE_NOT_SUPPORTED, "logits")
    refused(T(y, E((4,), f32)), L.ERR_INPUT_TYPE_NOT_SUPPORTED, "ids")
    refused(T(y, E((5,), np.int64)), L.ERR_WRONG_INPUT_SHAPE, "ids")
    refused(T(y, E((4, 1), np.int64)), L.ERR_WRONG_INPUT_SHAPE, "ids")
    refused(T(E((), f32), entropy=True), L.ERR_WRONG_INPUT_SHAPE, "logits")
    refused(T(E((4, 0), f32), entropy=True), L.ERR_NOT_SUPPORTED)
    for top in (-1, 51, 65):
        refused(T(y, ids, top=top), L.ERR_ATTRIBUTE_NOT_SUPPORTED, "top")
    refused(T(y), L.ERR_INVALID_ARGUMENT)
    refused(T(y, ids, out=(E((3,), f32),)), L.ERR_BUFFER_TOO_SMALL)
    row = hip.DeviceTensor.wrap(y.h.data, (4,), f32, 16, keepalive=y)
    refused(T(y, ids, out=(row,)), L.ERR_INVALID_ARGUMENT, "shares storage")
    one = E((4,), f32)
    refused(T(y, ids, entropy=True, out=(one, hip.DeviceTensor.wrap(one.h.data, (4,), f32, 16))), L.ERR_INVALID_ARGUMENT, "shares storage")
    lib, h = L.lib(), L.LxTensor()
    assert lib.lx_TokenLogProbs(ctypes.byref(y.h), None, 0, ctypes.byref(h), None, None, None) == L.ERR_INVALID_ARGUMENT
    assert lib.lx_TokenLogProbs(ctypes.byref(y.h), None, 3, None, None, ctypes.byref(h), None) == L.ERR_INVALID_ARGUMENT
    assert not h.data


def test_other_operators_refuse_the_8_bit_types(hip):
    from onnx_amd import _lib as L
    HIP = hip.HipExecutionProvider
    c = hip.DeviceTensor.empty((4, 8), E4M3)
    for r in (HIP.Add(c, c), HIP.Sqrt(c), HIP.Cast(c, L.FLOAT), HIP.Cast(hip.DeviceTensor.empty((4,), np.float32), E4M3),
              HIP.ReduceSum(c), HIP.ReduceMax(c), HIP.Softmax(c), HIP.MatMul(c, c), HIP.Transpose(c), HIP.Concat([c, c], 0),
              HIP.Gather(c, np.array([0])), HIP.Slice(c, [0], [1]), HIP.LayerNormDecomposed(c, c, c), HIP.GeluErf(c)):
        assert r.Status.name == "Failure" and r.Code in (L.ERR_INPUT_TYPE_NOT_SUPPORTED, L.ERR_NOT_SUPPORTED,
                                                         L.ERR_ATTRIBUTE_NOT_SUPPORTED), (r.Op, r.Code, r.Message)
