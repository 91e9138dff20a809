"""Performance cases of the scoring operators: block-scaled 8-bit floating point products (QuantizeBlocks, MatMulBlocks)
and the log-probabilities of tokens (TokenLogProbs), as a program calls them that scores texts with a vocabulary head.

listed() names the cases, draw() gives others of the same ranges.  With `own` false, run() computes the operators in
plain 32-bit torch; with `own` true it makes the HipExecutionProvider's calls, on torch allocations wrapped as
DeviceTensors.  exact() evaluates the definitions in 64 bits."""
import math

import torch

own = False

E4M3, E5M2 = 17, 19  # TensorElementType codes of Float8E4M3FN and Float8E5M2
TYPE = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
MANTISSA = {E4M3: 3, E5M2: 2}
LEAST = {E4M3: -6, E5M2: -14}  # exponent of the smallest normal value
BLOCK = 128


def listed():
    return [
        # One token's hidden state of a small encoder, quantised before its projection: the launch is the time.
        {"name": "quantize_1x384", "kind": "quantize", "rows": 1, "k": 384, "block_rows": 1, "to": E4M3},
        # Activations between the two feed-forward products, 8 documents of 512 tokens.
        {"name": "quantize_4096x1536", "kind": "quantize", "rows": 4096, "k": 1536, "block_rows": 1, "to": E4M3},
        # A vocabulary matrix quantised once, in 128x128 blocks, with the wider range of E5M2.
        {"name": "quantize_30522x768_blocks", "kind": "quantize", "rows": 30522, "k": 768, "block_rows": 128, "to": E5M2},
        # One token through a square projection of a large model: the weights are read once.
        {"name": "matmul_1x4096x4096", "kind": "matmul", "rows": 1, "k": 4096, "n": 4096, "b_rows": 128, "a": E4M3,
         "b": E4M3, "bias": False},
        # Four sequences padded to 197 tokens through a BERT-base projection, with its bias.
        {"name": "matmul_788x768x768", "kind": "matmul", "rows": 788, "k": 768, "n": 768, "b_rows": 128, "a": E4M3,
         "b": E4M3, "bias": True},
        # Odd sizes: rows that start at any byte, a last block of 73 columns, weights scaled row by row.
        {"name": "matmul_333x1225x1001_rows", "kind": "matmul", "rows": 333, "k": 1225, "n": 1001, "b_rows": 1, "a": E5M2,
         "b": E4M3, "bias": True},
        # 16 prompts of 512 tokens through a large model's feed-forward product.
        {"name": "matmul_8192x4096x8192", "kind": "matmul", "rows": 8192, "k": 4096, "n": 8192, "b_rows": 128, "a": E4M3,
         "b": E4M3, "bias": False},
        # The next token of one sequence: its candidates among a large vocabulary.
        {"name": "logprobs_1x131072_top20", "kind": "logprobs", "rows": 1, "vocab": 131072, "top": 20, "ids": "int64",
         "entropy": True},
        # The texts of a batch scored token by token (their probability under the model), padded rows among them.
        {"name": "logprobs_4096x30522", "kind": "logprobs", "rows": 4096, "vocab": 30522, "top": 0, "ids": "int64",
         "entropy": True},
        # A generating batch: each sequence's token, how sure the model was and what else it might have said.
        {"name": "logprobs_64x50001_top5", "kind": "logprobs", "rows": 64, "vocab": 50001, "top": 5, "ids": "int32",
         "entropy": True},
        # The head of a masked language model over the masked tokens of a batch: hidden states in, scores out.
        {"name": "head_512x768x30522", "kind": "head", "rows": 512, "k": 768, "n": 30522},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "quantize", "matmul", "matmul", "matmul", "logprobs", "logprobs", "logprobs", "head"])
    if kind == "quantize":
        k = rng.choice([384, 768, 1536, 4096, _size(rng, 1, 8192)])
        return {"kind": kind, "rows": _size(rng, 1, 33554432 // max(k, 1024)), "k": k, "block_rows": rng.choice([1, 1, 128]),
                "to": rng.choice([E4M3, E4M3, E5M2])}
    if kind == "matmul":
        k, n = (rng.choice([384, 768, 1536, 4096, 16 * _size(rng, 4, 512), _size(rng, 33, 8192)]) for _ in range(2))
        return {"kind": kind, "rows": _size(rng, 1, min(16384, (1 << 38) // (k * n))), "k": k, "n": n,
                "b_rows": rng.choice([1, 128, 128]), "a": rng.choice([E4M3, E4M3, E5M2]), "b": rng.choice([E4M3, E4M3, E5M2]),
                "bias": rng.random() < 0.5}
    if kind == "logprobs":
        v = rng.choice([30522, 32000, 131072, _size(rng, 100, 262144)])
        return {"kind": kind, "rows": _size(rng, 1, min(4096, 125000000 // v)), "vocab": v,
                "top": rng.choice([0, 1, 5, 20, _size(rng, 1, 64)]), "ids": rng.choice(["int32", "int64"]),
                "entropy": rng.random() < 0.7}
    return {"kind": kind, "rows": _size(rng, 1, 512), "k": rng.choice([384, 768, 1024]), "n": rng.choice([30522, _size(rng, 1000, 50000)])}


# ---- inputs ---------------------------------------------------------------------------------------------------
def _blocks(n):
    return -(-n // BLOCK)


def _weights(g, rows, k, b_rows, to, std):
    """A matrix as it is stored: codes [rows, k] and the scale of each block, for values around `std`."""
    scale = torch.rand(rows if b_rows == 1 else _blocks(rows), _blocks(k), device="cuda:0", generator=g)
    scale = (scale + 0.5) * (4 * std / LARGEST[to])
    codes = torch.randn(rows, k, device="cuda:0", generator=g) * (LARGEST[to] / 4)
    return codes.clamp_(-LARGEST[to], LARGEST[to]).to(TYPE[to]), scale


def _data(c, seed):
    """The inputs of a case as torch tensors by name."""
    g, k = torch.Generator(device="cuda:0"), c["kind"]
    g.manual_seed(seed)
    if k in ("quantize", "head"):
        # hidden states: a few channels are far larger than the others, which is what blocks are for
        x = torch.randn(c["rows"], c["k"], device="cuda:0", generator=g)
        x *= torch.exp(torch.randn(c["k"], device="cuda:0", generator=g))
        if k == "quantize":
            return {"x": x}
        w, ws = _weights(g, c["n"], c["k"], 128, E4M3, c["k"] ** -0.5)
        ids = torch.randint(0, c["n"], (c["rows"],), device="cuda:0", generator=g)
        return {"x": x, "b": w, "b_scale": ws, "bias": torch.randn(c["n"], device="cuda:0", generator=g) * 0.1,
                "ids": ids}
    if k == "matmul":
        d = {}
        d["a"], d["a_scale"] = _weights(g, c["rows"], c["k"], 1, c["a"], 1.0)
        d["b"], d["b_scale"] = _weights(g, c["n"], c["k"], c["b_rows"], c["b"], c["k"] ** -0.5)
        if c["bias"]:
            d["bias"] = torch.randn(c["n"], device="cuda:0", generator=g) * 0.1
        return d
    t, v = c["rows"], c["vocab"]
    x = torch.randn(t, v, device="cuda:0", generator=g) * 3
    # tokens that the model must not say are masked in every row; the last rows of a batch are padding
    x[:, torch.rand(v, device="cuda:0", generator=g) < 0.02] = -math.inf
    ids = torch.randint(0, v, (t,), device="cuda:0", generator=g)
    ids[t - t // 8:] = -1
    return {"x": x, "ids": ids.to(getattr(torch, c["ids"]))}


def prepare(case, seed):
    c, d = case, _data(case, seed)
    s = {"case": c, "in": d}
    if own:  # the tensors' handles and the outputs' storage, which a program keeps from call to call
        import onnx_amd
        onnx_amd.init(0)
        k, t = c["kind"], c["rows"]
        out = {}

        def new(name, *shape, dtype=torch.float32):
            out[name] = torch.empty(*shape, device="cuda:0", dtype=dtype)

        if k in ("quantize", "head"):
            b = c.get("block_rows", 1)
            new("q", t, c["k"], dtype=TYPE[c.get("to", E4M3)])
            new("s", -(-t // b), _blocks(c["k"]))
        if k in ("matmul", "head"):
            new("y", t, c["n"])
        if k in ("logprobs", "head"):
            new("lp", t)
            if c.get("entropy", True):
                new("h", t)
            if c.get("top", 0):
                new("top_ids", t, c["top"], dtype=torch.int64)
                new("top_lp", t, c["top"])
        s["out"] = out
        s["w"] = {n: onnx_amd.DeviceTensor.wrap_torch(x) for n, x in {**d, **out}.items()}
        torch.cuda.synchronize()
    return s


# ---- the framework's calls --------------------------------------------------------------------------------------
def _ok(r):
    if r.Code:
        raise RuntimeError(r.Message)


def _own(c, w, out):
    from onnx_amd import HipExecutionProvider as HIP

    k = c["kind"]
    if k in ("quantize", "head"):
        _ok(HIP.QuantizeBlocks(w["x"], to=c.get("to", E4M3), block_rows=c.get("block_rows", 1), out=(w["q"], w["s"])))
    if k == "matmul":
        _ok(HIP.MatMulBlocks(w["a"], w["a_scale"], w["b"], w["b_scale"], bias=w.get("bias"), out=w["y"]))
    if k == "head":
        _ok(HIP.MatMulBlocks(w["q"], w["s"], w["b"], w["b_scale"], bias=w["bias"], out=w["y"]))
    if k in ("logprobs", "head"):
        asked = [n for n in ("lp", "h", "top_ids", "top_lp") if n in w]
        _ok(HIP.TokenLogProbs(w["y" if k == "head" else "x"], w["ids"], top=c.get("top", 0), entropy="h" in w,
                              out=tuple(w[n] for n in asked)))
    if k == "head":
        return {n: out[n] for n in ("y", "lp", "h")}
    return out


# ---- the plain form -----------------------------------------------------------------------------------------------
def _to_grid(q, to):
    """64-bit values to the nearest of the 8-bit type, ties to even, beyond the largest to the largest."""
    e = torch.frexp(q)[1] - 1
    step = torch.ldexp(torch.ones_like(q), e.clamp(min=LEAST[to]) - MANTISSA[to])
    return (torch.round(q / step) * step).clamp(-LARGEST[to], LARGEST[to])


def _blocked(x, block_rows):
    """[rows, k] padded with zeros and seen as [row blocks, block_rows, k blocks, 128]."""
    r, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -r % block_rows))
    return x.reshape(-(-r // block_rows), block_rows, _blocks(k), BLOCK)


def _quantize(x, block_rows, to):
    r, k = x.shape
    b = _blocked(x, block_rows)
    amax = b.abs().amax((1, 3))
    # quotients in 64 bits: a 32-bit one next to the middle of two 8-bit values rounds onto it, and a scale in
    # another last bit moves values across such middles
    scale = torch.where(amax > 0, (amax.double() / LARGEST[to]).clamp(min=2.0 ** -126), 1.0).to(torch.float32)
    q = _to_grid(b.double() / scale.double()[:, None, :, None], to).to(torch.float32)
    return q.reshape(-1, q.shape[2] * BLOCK)[:r, :k].to(TYPE[to]), scale


def _values(codes, scale, b_rows, dtype):
    """The values that codes and their blocks' scales stand for."""
    r, k = codes.shape
    s = scale.to(dtype).repeat_interleave(b_rows, 0)[:r].repeat_interleave(BLOCK, 1)[:, :k]
    return codes.to(dtype) * s


def _product(a, a_scale, b, b_scale, bias, dtype):
    b_rows = 1 if b_scale.shape[0] == b.shape[0] else BLOCK
    y = torch.matmul(_values(a, a_scale, 1, dtype), _values(b, b_scale, b_rows, dtype).t())
    return y if bias is None else y + bias.to(dtype)


def _logprobs(x, ids, top, entropy):
    x = x.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total)
    at = ids.long()
    lp = (torch.gather(d, 1, at.clamp(0, x.shape[1] - 1)[:, None]) - lse)[:, 0]
    lp = torch.where(at < 0, 0.0, torch.where(at >= x.shape[1], math.nan, lp))
    got = {"lp": lp}
    if entropy:
        got["h"] = (lse - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / total)[:, 0]
    if top:
        v, i = torch.sort(d, dim=-1, descending=True, stable=True)
        got["top_ids"], got["top_lp"] = i[:, :top].contiguous(), v[:, :top] - lse
    return got


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(c, s["w"], s["out"])
    d, k = s["in"], c["kind"]
    if k == "quantize":
        q, scale = _quantize(d["x"], c["block_rows"], c["to"])
        return {"q": q, "s": scale}
    if k == "matmul":
        return {"y": _product(d["a"], d["a_scale"], d["b"], d["b_scale"], d.get("bias"), torch.float32)}
    if k == "logprobs":
        return _logprobs(d["x"], d["ids"], c["top"], c["entropy"])
    q, scale = _quantize(d["x"], 1, E4M3)
    y = _product(q, scale, d["b"], d["b_scale"], d["bias"], torch.float32)
    return {"y": y, **_logprobs(y, d["ids"], 0, True)}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c, k, t = case, case["kind"], case["rows"]
    if k == "quantize":
        return {"bytes": 5 * t * c["k"] + 4 * -(-t // c["block_rows"]) * _blocks(c["k"]), "flops": 2 * t * c["k"]}
    if k == "logprobs":
        top, w = c["top"], 4 if c["ids"] == "int32" else 8
        return {"bytes": 4 * t * c["vocab"] + t * (w + 4 + 4 * c["entropy"] + 12 * top), "flops": 5 * t * c["vocab"]}
    n, kb = c["n"], _blocks(c["k"])
    b_scales = n if c.get("b_rows") == 1 else _blocks(n)
    product = n * c["k"] + 4 * kb * b_scales + 4 * t * n + 4 * n * c.get("bias", True)
    if k == "matmul":
        return {"bytes": product + t * (c["k"] + 4 * kb), "flops": 2 * t * n * c["k"]}
    return {"bytes": product + 4 * t * c["k"] + 16 * t, "flops": 2 * t * n * c["k"] + 5 * t * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _codes64(x, rows, to):
    """Codes (as values) and scales by the definition, the codes by search among the type's own values."""
    r, k = x.shape
    grid = torch.arange(256, dtype=torch.uint8, device=x.device).view(TYPE[to]).double()
    grid = torch.sort(grid[torch.isfinite(grid) & (grid >= 0)])[0].unique()  # 0, ..., the largest
    p = torch.zeros(-(-r // rows) * rows, _blocks(k) * BLOCK, device=x.device, dtype=torch.float32)
    p[:r, :k] = x
    p = p.reshape(-1, rows, _blocks(k), BLOCK).permute(0, 2, 1, 3)
    top = p.abs().reshape(p.shape[0], p.shape[1], -1).max(-1)[0].double()
    scale = torch.where(top > 0, torch.maximum(top / LARGEST[to], torch.full_like(top, 2.0 ** -126)), 1.0)
    v = p.double() / scale.float().double()[:, :, None, None]
    i = torch.searchsorted(grid, v.abs().contiguous()).clamp(1, len(grid) - 1)
    low, high = v.abs() - grid[i - 1], grid[i] - v.abs()
    # the grid's even places are the codes with an even last bit: ties go there
    up = (high < low) | ((high == low) & (i % 2 == 0))
    c = torch.copysign(torch.where(up, grid[i], grid[i - 1]), v)
    return c.permute(0, 2, 1, 3).reshape(p.shape[0] * rows, -1)[:r, :k], scale


def _product64(a, a_scale, b, b_scale, bias):
    """Block by block of the inner axis, the blocks' sums scaled as the definition scales them."""
    r, k = a.shape
    n = b.shape[0]
    cols = torch.arange(n, device=a.device) // (1 if b_scale.shape[0] == n else BLOCK)
    y = torch.zeros(r, n, device=a.device, dtype=torch.float64)
    for j in range(_blocks(k)):
        part = a[:, j * BLOCK:(j + 1) * BLOCK].double() @ b[:, j * BLOCK:(j + 1) * BLOCK].double().t().contiguous()
        y += part * a_scale[:, j, None].double() * b_scale[cols, j].double()
    return y if bias is None else y + bias.double()


def _logprobs64(x, ids, top, entropy):
    """Row ranges at a time (a 64-bit copy of the whole would be large)."""
    parts = []
    for r in range(0, x.shape[0], 512):
        v, at = x[r:r + 512].double(), ids[r:r + 512].long()
        lse = torch.logsumexp(v, -1)
        p = torch.exp(v - lse[:, None])
        said = v[torch.arange(len(at), device=v.device), at.clamp(0, v.shape[1] - 1)] - lse
        got = {"lp": torch.where(at < 0, torch.zeros_like(said), torch.where(at < v.shape[1], said, math.nan))}
        if entropy:
            got["h"] = -torch.xlogy(p, p).sum(-1)
        if top:
            order = torch.sort(v, dim=-1, descending=True, stable=True)
            got["top_ids"], got["top_lp"] = order[1][:, :top], order[0][:, :top] - lse[:, None]
        parts.append(got)
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}


def exact(case, seed):
    c, d = case, _data(case, seed)
    k = c["kind"]
    if k == "quantize":
        q, s = _codes64(d["x"], c["block_rows"], c["to"])
        return {"q": q, "s": s}
    if k == "matmul":
        return {"y": _product64(d["a"], d["a_scale"], d["b"], d["b_scale"], d.get("bias"))}
    if k == "logprobs":
        return _logprobs64(d["x"], d["ids"], c["top"], c["entropy"])
    q, s = _codes64(d["x"], 1, E4M3)
    y = _product64(q, s.float(), d["b"], d["b_scale"], d["bias"])
    return {"y": y, **_logprobs64(y, d["ids"], 0, True)}
