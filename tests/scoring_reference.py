"""The scoring operators (QuantizeBlocks, MatMulBlocks, TokenLogProbs) in plain numpy and 64 bits, from their
definitions, with bounds on what float32 sums may differ by.  Float8 codes are bytes."""
import numpy as np

E4M3, E5M2 = 17, 19
MAX = {E4M3: 448.0, E5M2: 57344.0}
U = 2.0 ** -24  # half a step of float32


def _decode_table(fmt):
    m, bias = (3, 7) if fmt == E4M3 else (2, 15)
    c = np.arange(256)
    e, f, sign = (c & 127) >> m, (c & ((1 << m) - 1)) / (1 << m), np.where(c & 128, -1.0, 1.0)
    v = np.where(e == 0, f * 2.0 ** (1 - bias), (1 + f) * 2.0 ** (e - bias)) * sign
    if fmt == E4M3:
        v[[0x7f, 0xff]] = np.nan
    else:
        v[[0x7c, 0xfc]] = [np.inf, -np.inf]
        v[[0x7d, 0x7e, 0x7f, 0xfd, 0xfe, 0xff]] = np.nan
    return v


VALUES = {f: _decode_table(f) for f in (E4M3, E5M2)}


def decode(codes, fmt):
    return VALUES[fmt][codes]


def blocks(n):
    return -(-n // 128)


def in_float(v):
    """Values that float32 has no room for are infinite in it: from half a step above its largest on (largest minus
    lowest, twice the largest, is one)."""
    beyond = np.abs(v) >= float(np.finfo(np.float32).max) * (1 + U / 2)
    return np.where(beyond, np.copysign(np.inf, v), v)


def quantize(x, fmt, block_rows):
    """(values of the codes, float32 scales) of x [..., N, K] (or [K])."""
    x = np.asarray(x, np.float32)
    lead = x.shape[:-2] if x.ndim >= 2 else ()
    n, k = (x.shape[-2], x.shape[-1]) if x.ndim >= 2 else (1, x.shape[-1])
    v = x.reshape((-1, n, k))
    pad = np.zeros((v.shape[0], -(-n // block_rows) * block_rows, blocks(k) * 128), np.float32)
    pad[:, :n, :k] = v
    b = pad.reshape(v.shape[0], -1, block_rows, blocks(k), 128).transpose(0, 1, 3, 2, 4)
    finite = np.where(np.isfinite(b), np.abs(b), 0)
    amax = finite.max((3, 4)).astype(np.float64)
    scale = np.where(amax > 0, np.maximum(amax / MAX[fmt], 2.0 ** -126), 1.0).astype(np.float32)
    q = b.astype(np.float64) / scale.astype(np.float64)[..., None, None]
    grid = VALUES[fmt][:128]
    grid = grid[np.isfinite(grid)]  # ascending, index = code
    a = np.minimum(np.abs(q), MAX[fmt])
    a = np.where(np.isnan(q), 0, a)
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    up, down = grid[hi] - a, a - grid[hi - 1]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    val = np.where(np.isnan(q), np.nan, np.copysign(grid[code], q))
    val = val.transpose(0, 1, 3, 2, 4).reshape(pad.shape)[:, :n, :k].reshape(x.shape)
    shape = lead + ((scale.shape[1],) if x.ndim >= 2 else ()) + (blocks(k),)
    return val, scale.reshape(shape)


def matmul(a, sa, b, sb, bias=None):
    """(product, bound on a float32 evaluation's error) of code values a [M, K], b [N, K] with their scales."""
    (m, k), n = a.shape, b.shape[0]
    rows = np.arange(n) if sb.shape[0] == n else np.arange(n) // 128
    y, mag = np.zeros((m, n)), np.zeros((m, n))
    for j in range(blocks(k)):
        s = sa[:, j, None].astype(np.float64) * sb[rows, j].astype(np.float64)
        ab, bb = a[:, 128 * j:128 * (j + 1)], b[:, 128 * j:128 * (j + 1)]
        y += (ab @ bb.T) * s
        mag += (np.abs(ab) @ np.abs(bb).T) * np.abs(s)
    # 128 float32 additions a block (a step each: the matrix unit may truncate), the scales' product, its product
    # with the block's sum and one addition a block; each partial sum is at most the sum of the magnitudes
    err = (2 * 128 + blocks(k) + 3) * U * mag
    if bias is not None:
        y = y + bias.astype(np.float64)
        err = err + U * (np.abs(y) + err)
    return y, err + 1e-37


def logprobs(x, ids=None, top=0):
    """64-bit results by name, and bounds (`*_err`) on a float32 evaluation's errors, of logits x [T, V]."""
    x = np.asarray(x, np.float32)
    t, v = x.shape
    with np.errstate(all="ignore"):
        d = x.astype(np.float64)
        m = d.max(-1, keepdims=True)
        z = np.where(np.isneginf(d), -np.inf, d - m)
        e = np.exp(z)
        s = e.sum(-1, keepdims=True)
        bad = ~np.isfinite(m[:, 0]) | np.isnan(d).any(-1)
        lse = np.log(s)
        p = e / s
        away = np.where(e > 0, -z, 0.0)
        h = (lse + (p * away).sum(-1, keepdims=True))[:, 0]
        # relative error of a term: the difference's rounding, the factor log2(e)'s and the product's (three of |z|
        # half steps) and the exponential's own (two steps); then the additions of a sum in parts: at most V / 512
        # terms after each other and about 64 merges, each of which rounds three times
        rel = U * (3 * away + 4)
        adds = U * (v / 512 + 3 * 64 + 64)
        ls_err = (p * rel).sum(-1) + adds + U * (np.abs(lse[:, 0]) + 1) * 2
        # the second sum: its terms' second factor rounds once more
        mean = (p * away).sum(-1)
        h_err = ls_err + (p * away * (rel + 2 * U)).sum(-1) + mean * (2 * adds + ls_err) + 4 * U * (np.abs(h) + mean)
        got = {"h": np.where(bad, np.nan, h), "h_err": h_err}
        if ids is not None:
            ids = np.asarray(ids, np.int64)
            zi = z[np.arange(t), np.clip(ids, 0, v - 1)]
            lp = np.where(bad, np.nan, zi - lse[:, 0])
            lp = np.where(ids < 0, 0.0, np.where(ids >= v, np.nan, lp))
            got["lp"], got["lp_err"] = in_float(lp), ls_err + U * (np.abs(np.where(np.isfinite(zi), zi, 0)) + np.abs(np.where(np.isfinite(lp), lp, 0)))
        if top:
            # NaN last; equal logits by index
            order = np.argsort(np.where(np.isnan(d), -np.inf, d) * -1, axis=-1, kind="stable")
            nan_last = np.take_along_axis(np.isnan(d), order, -1)
            order = np.take_along_axis(order, np.argsort(nan_last, axis=-1, kind="stable"), -1)[:, :top]
            zt = np.take_along_axis(z, order, -1)
            got["top_ids"] = order
            got["top_lp"] = in_float(np.where(bad[:, None], np.nan, zt - lse))
            got["top_lp_err"] = ls_err[:, None] + 2 * U * (np.abs(np.where(np.isfinite(zt), zt, 0)) + np.abs(lse))
    return got
