"""Expert routing and the block-128 FP8 operators as cases that can be timed.

Six operators, each over the range of sizes that it is called with:

  route         router logits -> expert ids and weights: softmax or sigmoid scores, a balancing bias
                that takes part in the choice only, groups of experts, renormalised weights
  route_train   the same and the gradient of the logits from the gradient of the weights
  quant         activations (or SiLU(gate) * up of them) -> e4m3 values with one fp32 scale per row and
                128 columns; whole batches, or the rows of row-concatenated groups
  quant_weight  weights -> e4m3 values with one fp32 scale per 128 x 128 block
  gemm          (m, k) x (n, k) of such operands
  grouped       the same for each group of a row-concatenated batch and its own weights

Scales of activations are held by 128-column block: (ceil(k / 128), rows rounded up to 4).  Values in 8
bits are returned as float8_e4m3fn.  A case is a dict of plain values.
"""

from __future__ import annotations

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3 = torch.float8_e4m3fn
_TINY = 2.0 ** -126      # the smallest scale


# ---- the cases ---------------------------------------------------------------------------


def listed():
    return [
        # a decode step of 16 sequences: 256 experts in 8 groups of which 4 take part, sigmoid scores, balancing bias
        dict(name="route_decode", path="route", tokens=16, experts=256, topk=8, score="sigmoid", bias=True, groups=8,
             topk_groups=4, group_top=2, renormalize=True, scale=2.5, dtype="f32"),
        # the prefill that the routed layer's benchmark runs, with the same router
        dict(name="route_prefill", path="route", tokens=8192, experts=256, topk=8, score="sigmoid", bias=True, groups=8,
             topk_groups=4, group_top=2, renormalize=True, scale=2.5, dtype="f32"),
        # a training micro-batch of odd length: softmax over 160 experts, groups by their best expert, weights as they are
        dict(name="route_train_softmax", path="route_train", tokens=16383, experts=160, topk=6, score="softmax", bias=False,
             groups=8, topk_groups=3, group_top=1, renormalize=False, scale=16.0, dtype="bf16"),
        # fine-tuning on a short sequence: a small layer whose expert count is no multiple of anything
        dict(name="route_train_short", path="route_train", tokens=333, experts=61, topk=4, score="sigmoid", bias=True,
             groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0, dtype="f32"),
        # the hidden states of a decode step on their way into a projection
        dict(name="quant_decode", path="quant", groups=0, lo=16, hi=16, rows_seed=0, k=7168, silu=False, dtype="bf16"),
        # between the two products of an expert layer: SiLU(gate) * up of the rows of 64 ragged groups
        dict(name="quant_silu_groups", path="quant", groups=64, lo=160, hi=352, rows_seed=1, k=2048, silu=True, dtype="bf16"),
        # the first projections of 16 experts when a checkpoint is loaded
        dict(name="quant_weight_experts", path="quant_weight", l=16, n=4096, k=7168, dtype="bf16"),
        # one small matrix with ragged edges, kept in fp32 by its trainer
        dict(name="quant_weight_odd", path="quant_weight", l=1, n=1048, k=3088, dtype="f32"),
        # a decode step through a down projection: the weights stream past a few rows
        dict(name="gemm_decode", path="gemm", m=16, n=7168, k=2048, out="bf16"),
        # a prefill through an up projection, its length no round number
        dict(name="gemm_prefill", path="gemm", m=4101, n=7168, k=4096, out="bf16"),
        # a decode step through 64 experts, some of them without a row
        dict(name="grouped_decode", path="grouped", groups=64, lo=0, hi=16, rows_seed=2, n=4096, k=7168, scaled=False, out="bf16"),
        # a prefill through the second projection: 256 rows an expert, more or less, weighted by the router
        dict(name="grouped_prefill", path="grouped", groups=64, lo=208, hi=304, rows_seed=3, n=7168, k=2048, scaled=True, out="bf16"),
    ]


def _rows(case):
    """Rows of each group (no groups: of the whole batch): part of the case, so that every state of it
    does the same work."""
    if not case["groups"]:
        return [case["hi"]]
    g = torch.Generator().manual_seed(case["rows_seed"])
    return torch.randint(case["lo"], case["hi"] + 1, (case["groups"],), generator=g).tolist()


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + step)))
    return max(lo, min(hi, int(v) // step * step))


#: the largest listed case in each resource; drawn cases stay under it
_MAX_FLOPS = 4.9e11
_MAX_BYTES = 1.45e9


def draw(rng):
    while True:
        path = rng.choice(["route", "route_train", "quant", "quant_weight", "gemm", "grouped"])
        if path in ("route", "route_train"):
            groups = rng.choice([1, 1, 1, 2, 4, 8, 16])
            per = max(1, _log(rng, 8, 512) // groups)
            topk_groups = rng.randint(1, groups)
            case = dict(path=path, tokens=_log(rng, 1, 16384), experts=groups * per,
                        topk=min(rng.choice([1, 2, 4, 6, 8, 10]), topk_groups * per), score=rng.choice(["softmax", "sigmoid"]),
                        bias=rng.random() < 0.5, groups=groups, topk_groups=topk_groups,
                        group_top=rng.randint(1, min(2, per)), renormalize=rng.random() < 0.6,
                        scale=rng.choice([1.0, 1.0, 2.5, 16.0]), dtype=rng.choice(["f32", "bf16", "fp16"]))
        elif path == "quant":
            groups = _log(rng, 2, 64) if rng.random() < 0.5 else 0
            hi = _log(rng, 4, 512) if groups else _log(rng, 1, 16384)
            case = dict(path=path, groups=groups, lo=hi // 8 if groups else hi, hi=hi, rows_seed=rng.randrange(1 << 20),
                        k=_log(rng, 64, 7168, 16), silu=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16", "f32"]))
        elif path == "quant_weight":
            case = dict(path=path, l=_log(rng, 1, 16), n=_log(rng, 64, 8192, 8), k=_log(rng, 64, 7168, 16),
                        dtype=rng.choice(["bf16", "fp16", "f32"]))
        elif path == "gemm":
            case = dict(path=path, m=_log(rng, 1, 8192), n=_log(rng, 64, 8192, 8), k=_log(rng, 64, 7168, 16),
                        out=rng.choice(["bf16", "bf16", "fp16", "f32"]))
        else:
            hi = _log(rng, 4, 640)
            case = dict(path=path, groups=_log(rng, 2, 64), lo=hi // 8, hi=hi, rows_seed=rng.randrange(1 << 20),
                        n=_log(rng, 128, 7168, 8), k=_log(rng, 128, 7168, 16), scaled=rng.random() < 0.5,
                        out=rng.choice(["bf16", "bf16", "fp16", "f32"]))
        w = work(case)
        if w["flops"] <= _MAX_FLOPS and w["bytes"] <= _MAX_BYTES and (path not in ("quant", "grouped") or sum(_rows(case))):
            return case


# ---- the work that cannot be left out ------------------------------------------------------


_SIZE = {"f32": 4.0, "bf16": 2.0, "fp16": 2.0}


def work(case):
    p = case["path"]
    if p in ("route", "route_train"):
        t, e, k = case["tokens"], case["experts"], case["topk"]
        logits, picks = t * e * _SIZE[case["dtype"]], t * k * 8.0
        if p == "route":
            return {"bytes": logits + picks + (4.0 * e if case["bias"] else 0.0), "flops": 4.0 * t * e}
        # logits in, ids and weights out, the gradient of the weights in, that of the logits out
        return {"bytes": 2 * logits + picks + 4.0 * t * k + (4.0 * e if case["bias"] else 0.0), "flops": 8.0 * t * e}
    if p == "quant":
        rows, k = sum(_rows(case)), case["k"]
        x = rows * k * _SIZE[case["dtype"]] * (2 if case["silu"] else 1)
        return {"bytes": x + rows * k + 4.0 * rows * -(-k // 128), "flops": rows * k * (8.0 if case["silu"] else 3.0)}
    if p == "quant_weight":
        l, n, k = case["l"], case["n"], case["k"]
        return {"bytes": l * n * k * (_SIZE[case["dtype"]] + 1.0) + 4.0 * l * -(-n // 128) * -(-k // 128), "flops": 3.0 * l * n * k}
    n, k = case["n"], case["k"]
    rows = _rows(case) if p == "grouped" else [case["m"]]
    total, used = sum(rows), sum(r > 0 for r in rows)
    return {"bytes": total * (k + 4.0 * -(-k // 128)) + used * (n * k + 4.0 * -(-n // 128) * -(-k // 128)) +
            total * n * _SIZE[case["out"]] + (4.0 * total if case.get("scaled") else 0.0),
            "flops": 2.0 * total * n * k}


# ---- inputs --------------------------------------------------------------------------------


def _offsets(rows):
    """Start of each group, a multiple of 128, and the rows that all of them take."""
    offs, at = [], 0
    for r in rows:
        offs.append(at)
        at += -(-r // 128) * 128
    return offs, max(at, 128)


def _activations(g, rows, k, dtype):
    """Hidden states: rows of different size, a few columns that stand out."""
    x = torch.randn((rows, k), device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn((rows, 1), device="cuda", generator=g))
    x *= torch.where(torch.rand((1, k), device="cuda", generator=g) < 0.002, 20.0, 1.0)
    return x.to(dtype)


def _weights(g, l, n, k, dtype):
    w = torch.empty((l, n, k), dtype=dtype, device="cuda")
    for i in range(l):
        w[i] = 0.02 * torch.randn((n, k), device="cuda", generator=g)
    return w


def _blocks(x, size):
    """Columns in blocks of `size`, the last one filled up with zeros."""
    k = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -k % size)).unflatten(-1, (-1, size))


def _quantized_rows(x):
    """Operands as they reach a product: (rows, k) e4m3 bytes, (k blocks, rows rounded up to 4) scales."""
    rows, k = x.shape
    b = _blocks(x.float(), 128)
    s = (b.abs().amax(-1) / 448.0).clamp(min=_TINY)
    q = (b / s[..., None]).flatten(-2)[:, :k].to(_E4M3)
    return q.contiguous().view(torch.uint8), torch.nn.functional.pad(s.t(), (0, -rows % 4)).contiguous()


def _quantized_weights(g, l, n, k):
    q = torch.empty((l, n, k), dtype=torch.uint8, device="cuda")
    s = torch.empty((l, -(-n // 128), -(-k // 128)), device="cuda")
    for i in range(l):
        w = _weights(g, 1, n, k, torch.float32)[0]
        s[i] = (_blocks(_blocks(w, 128).abs().amax(-1).t(), 128).amax(-1).t() / 448.0).clamp(min=_TINY)
        q[i] = (w / _expanded(s[i], n, k)).to(_E4M3).view(torch.uint8)
    return q, s


def _expanded(s, n, k):
    """One value per block -> one per element."""
    return s.repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    p, i32 = case["path"], dict(dtype=torch.int32, device="cuda")
    s = dict(case)
    if p in ("route", "route_train"):
        t, e = case["tokens"], case["experts"]
        s["logits"] = (1.5 * torch.randn((t, e), device="cuda", generator=g)).to(_TYPES[case["dtype"]])
        s["bias"] = 0.1 * torch.randn((e,), device="cuda", generator=g) if case["bias"] else None
        if p == "route_train":
            s["grad"] = torch.randn((t, case["topk"]), device="cuda", generator=g)
        return s
    if p == "quant_weight":
        s["w"] = _weights(g, case["l"], case["n"], case["k"], _TYPES[case["dtype"]])
        return s
    k = case["k"]
    if p == "gemm":
        s["a_q"], s["a_sf"] = _quantized_rows(_activations(g, case["m"], k, torch.float32))
        s["b_q"], s["b_sf"] = (t[0] for t in _quantized_weights(g, 1, case["n"], k))
        return s
    s["rows"] = rows = _rows(case)
    offs, total = _offsets(rows)
    if case["groups"]:
        s["offsets"], s["group_rows"] = torch.tensor(offs, **i32), torch.tensor(rows, **i32)
    else:
        total = rows[0]
    s["total"] = total
    if p == "quant":
        s["x"] = _activations(g, total, k * (2 if case["silu"] else 1), _TYPES[case["dtype"]])
        # the program's buffers: rows that belong to no group stay as they are
        s["q"] = torch.zeros((total, k), dtype=torch.uint8, device="cuda")
        s["sf"] = torch.zeros((-(-k // 128), -(-total // 4) * 4), device="cuda")
        return s
    s["a_q"], s["a_sf"] = _quantized_rows(_activations(g, total, k, torch.float32))
    s["b_q"], s["b_sf"] = _quantized_weights(g, len(rows), case["n"], k)
    s["row_scale"] = torch.rand((total,), device="cuda", generator=g) if case["scaled"] else None
    s["y"] = torch.zeros((total, case["n"]), dtype=_TYPES[case["out"]], device="cuda")
    return s


# ---- one pass ------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    p = s["path"]
    if p == "route":
        ids, weights, _, _ = _route(s)
        return ids, weights
    if p == "route_train":
        return _route_train(s)
    if p == "quant":
        return _quant(s)
    if p == "quant_weight":
        return _quant_weight(s)
    if p == "gemm":
        return (_dequantized_rows(s) @ _dequantized_weights(s).t()).to(_TYPES[s["out"]])
    return _grouped(s)


def _run_own(s):
    from mosaicist_b200 import ops

    p = s["path"]
    if p in ("route", "route_train"):
        kind = dict(score=s["score"], renormalize=s["renormalize"], scale=s["scale"])
        ids, weights = ops.moe_route(s["logits"], s["topk"], bias=s["bias"], groups=s["groups"], topk_groups=s["topk_groups"],
                                     group_top=s["group_top"], **kind)
        if p == "route":
            return ids, weights
        return ids, weights, ops.moe_route_backward(s["grad"], s["logits"], ids, weights, **kind)
    if p == "quant":
        q, sf = ops.quantize_fp8_block(s["x"], silu=s["silu"], group_offsets=s.get("offsets"), group_rows=s.get("group_rows"),
                                       out=(s["q"], s["sf"]))
        return q.view(_E4M3), sf
    if p == "quant_weight":
        q, sf = ops.quantize_fp8_block_weight(s["w"])
        return q.view(_E4M3), sf
    if p == "gemm":
        return ops.gemm_fp8_block(s["a_q"], s["a_sf"], s["b_q"], s["b_sf"], out_dtype=_TYPES[s["out"]])
    return ops.ragged_grouped_gemm_fp8_block(s["a_q"], s["a_sf"], s["b_q"], s["b_sf"], s["offsets"], s["group_rows"],
                                             row_scale=s["row_scale"], out=s["y"])


# The plain forms.  Scores are compared with one another, so they are computed in 64 bits.


def _route(s):
    x = s["logits"].double()
    if s["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    key = score if s["bias"] is None else score + s["bias"].double()
    if s["groups"] > 1:
        by = key.unflatten(-1, (s["groups"], -1))
        best = by.sort(dim=-1, descending=True, stable=True).values[..., :s["group_top"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :s["topk_groups"]]
        allowed = torch.zeros_like(best, dtype=torch.bool).scatter(-1, kept, True)
        key = torch.where(allowed[..., None], by, -torch.inf).flatten(-2)
    ids = key.sort(dim=-1, descending=True, stable=True).indices[:, :s["topk"]]
    picked = score.gather(-1, ids)
    share = picked / picked.sum(-1, keepdim=True) if s["renormalize"] else picked
    return ids.int(), (share * s["scale"]).float(), score, share


def _route_train(s):
    ids, weights, score, share = _route(s)
    at, g = ids.long(), s["grad"].double() * s["scale"]
    picked = score.gather(-1, at)
    # to the picked scores, then through the scores to the logits
    if s["renormalize"]:
        g = (g - (g * share).sum(-1, keepdim=True)) / picked.sum(-1, keepdim=True)
    to_score = torch.zeros_like(score).scatter(-1, at, g)
    if s["score"] == "softmax":
        grad = score * (to_score - (to_score * score).sum(-1, keepdim=True))
    else:
        grad = to_score * score * (1.0 - score)
    return ids, weights, grad.to(s["logits"].dtype)


def _group_rows_index(s):
    """Rows of every group side by side (groups, longest), and which of them exist."""
    r = torch.arange(max(s["rows"]), device="cuda")
    there = r < s["group_rows"][:, None]
    return torch.where(there, s["offsets"][:, None] + r, 0), there


def _quant(s):
    x, k = s["x"].float(), s["k"]
    if s["silu"]:
        gate, up = x[:, :k], x[:, k:]
        x = gate / (1.0 + torch.exp(-gate)) * up
    b = _blocks(x, 128)
    scale = (b.abs().amax(-1) / 448.0).clamp(min=_TINY)
    q = (b / scale[..., None]).flatten(-2)[:, :k].to(_E4M3).view(torch.uint8)
    sf = torch.nn.functional.pad(scale.t(), (0, s["sf"].shape[1] - s["total"]))
    if s["groups"]:
        at, there = _group_rows_index(s)
        live = torch.zeros(s["sf"].shape[1], dtype=torch.bool, device="cuda").index_fill(0, at[there], True)
        q = torch.where(live[:s["total"], None], q, s["q"])
        sf = torch.where(live, sf, s["sf"])
    return q.view(_E4M3), sf


def _quant_weight(s):
    w = s["w"].float()
    tiles = _blocks(_blocks(w, 128).abs().amax(-1).transpose(-1, -2), 128).amax(-1).transpose(-1, -2)
    sf = (tiles / 448.0).clamp(min=_TINY).contiguous()
    return (w / _expanded(sf, s["n"], s["k"])).to(_E4M3), sf


def _dequantized_rows(s):
    a = s["a_q"].view(_E4M3).float()
    return a * s["a_sf"].t()[:a.shape[0]].repeat_interleave(128, -1)[:, :a.shape[1]]


def _dequantized_weights(s):
    return s["b_q"].view(_E4M3).float() * _expanded(s["b_sf"], s["n"], s["k"])


def _grouped(s):
    at, there = _group_rows_index(s)
    a = _dequantized_rows(s)
    if s["row_scale"] is not None:
        a = a * s["row_scale"][:, None]
    y = a[at] @ _dequantized_weights(s).transpose(-1, -2)
    return s["y"].index_copy(0, at[there], y[there].to(s["y"].dtype))


# ---- the definition, in 64 bits ------------------------------------------------------------


def _e4m3(x):
    """The nearest e4m3 value, ties to even: 4 significant bits down to an exponent of -6, 448 at most."""
    mag = x.abs().clamp(max=448.0)
    step = torch.exp2((torch.frexp(mag).exponent - 1).clamp(min=-6).double() - 3)
    return torch.copysign(torch.round(mag / step) * step, x)


def _scale64(amax):
    return torch.clamp((amax / 448.0).float(), min=_TINY).double()


def exact(case, seed):
    s = prepare(case, seed)
    p = case["path"]
    if p in ("route", "route_train"):
        return _exact_route(case, s)
    if p == "quant":
        return _exact_quant(case, s)
    k = case["k"]
    if p == "quant_weight":
        qs, sfs = [], []
        for w in s["w"]:
            q, sf = torch.empty(w.shape, dtype=torch.float64, device="cuda"), []
            for r in range(0, case["n"], 128):
                part = w[r:r + 128].double()
                sf.append(torch.stack([_scale64(part[:, c:c + 128].abs().max()) for c in range(0, k, 128)]))
                q[r:r + 128] = _e4m3(part / sf[-1].repeat_interleave(128)[:k])
            qs.append(q.float())
            sfs.append(torch.stack(sf))
        return torch.stack(qs), torch.stack(sfs)
    if p == "gemm":
        return _exact_product(s["a_q"], s["a_sf"][:, :case["m"]], s["b_q"], s["b_sf"])
    y = torch.zeros((s["total"], case["n"]), dtype=torch.float64, device="cuda")
    for g, (o, r) in enumerate(zip(s["offsets"].tolist(), s["rows"])):
        if r:
            y[o:o + r] = _exact_product(s["a_q"][o:o + r], s["a_sf"][:, o:o + r], s["b_q"][g], s["b_sf"][g])
            if case["scaled"]:
                y[o:o + r] *= s["row_scale"][o:o + r, None].double()
    return y


def _exact_product(a_q, a_sf, b_q, b_sf):
    """The sum over 128-column blocks of their products, each times its two scales."""
    m, k = a_q.shape
    n = b_q.shape[0]
    y = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    of_row = torch.arange(n, device="cuda") // 128
    for c in range(a_sf.shape[0]):
        a = a_q[:, 128 * c:128 * c + 128].contiguous().view(_E4M3).double() * a_sf[c].double()[:, None]
        b = b_q[:, 128 * c:128 * c + 128].contiguous().view(_E4M3).double() * b_sf[:, c].double()[of_row][:, None]
        y.addmm_(a, b.t())
    return y


def _exact_quant(case, s):
    k = case["k"]
    q = torch.zeros((s["total"], k), dtype=torch.float64, device="cuda")
    sf = torch.zeros(s["sf"].shape, dtype=torch.float64, device="cuda")
    offs = s["offsets"].tolist() if case["groups"] else [0]
    for o, r in zip(offs, s["rows"]):
        x = s["x"][o:o + r].double()
        if case["silu"]:
            x = x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:]
        for c in range(0, k, 128):
            part = x[:, c:c + 128]
            if r:
                scale = _scale64(part.abs().amax(1))
                sf[c // 128, o:o + r] = scale
                q[o:o + r, c:c + 128] = _e4m3(part / scale[:, None])
    return q, sf


def _exact_route(case, s):
    x, t = s["logits"].double(), case["tokens"]
    score = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
    key = score.clone() if s["bias"] is None else score + s["bias"].double()
    rows = torch.arange(t, device="cuda")
    per = case["experts"] // case["groups"]
    if case["groups"] > 1:
        strength = torch.stack([key[:, i * per:(i + 1) * per].topk(case["group_top"]).values.sum(1) for i in range(case["groups"])], 1)
        barred = torch.ones_like(strength, dtype=torch.bool)
        for _ in range(case["topk_groups"]):
            best = strength.argmax(1)
            barred[rows, best] = False
            strength[rows, best] = -torch.inf
        key[barred.repeat_interleave(per, 1)] = -torch.inf
    ids = []
    for _ in range(case["topk"]):
        top = key.amax(1, keepdim=True)
        ids.append(torch.where(key == top, torch.arange(case["experts"], device="cuda"), case["experts"]).amin(1))
        key[rows, ids[-1]] = -torch.inf
    ids = torch.stack(ids, 1)
    picked = score.gather(1, ids)
    total = picked.sum(1, keepdim=True) if case["renormalize"] else 1.0
    weights = picked / total * case["scale"]
    if case["path"] == "route":
        return ids.int(), weights
    # d weights[i] / d score[j] = scale (delta_ij - weights[i] / scale) / total where renormalised, scale delta_ij otherwise;
    # d score[i] / d logits[j] = score[i] (delta_ij - score[j]) for softmax, delta_ij score (1 - score) for sigmoid
    g = s["grad"].double() * case["scale"]
    if case["renormalize"]:
        g = (g - (g * picked).sum(1, keepdim=True) / total) / total
    if case["score"] == "sigmoid":
        grad = torch.zeros_like(score).scatter_add(1, ids, g * picked * (1.0 - picked))
    else:
        grad = -score * (g * picked).sum(1, keepdim=True)
        grad = grad.scatter_add(1, ids, g * picked)
    return ids.int(), weights, grad
