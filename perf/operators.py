"""Cases for the operators around the attention block: RMS norm with the
residual's addition (output in 16/32 bits, or in e4m3 with one scale per 128
values), quantisation to e4m3, the block-scaled e4m3 matrix product, and token
sampling.

`run` computes an operator in elementary torch operations, or, with `own` set,
through the framework's entry points.  Sizes are those of the decode workloads'
models (hidden 2048, 4096, 8192; vocabularies 32000 and 128256), batches from
one token to prefill chunks, and odd ones.
"""
import math
import os
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0
TINY = 2.0 ** -126  # the smallest scale: an all-zero group
DEV = "cuda"


def _lib():
    if "cottus_b200" not in sys.modules:  # the package's folder is not importable by its own name
        sys.path.insert(0, os.path.join(os.getcwd(), "cottus-runtime_b200"))
        import cottus_b200  # noqa: F401
    return sys.modules["cottus_b200"]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one token of a 2048-wide model: the norm before its attention block (fp16 activations)
        dict(name="norm_1x2048_f16", op="norm", rows=1, hidden=2048, x="f32", residual=False, out="f16"),
        # a decode batch of a 4096-wide model, ahead of an 8-bit projection
        dict(name="norm_64x4096_e4m3", op="norm", rows=64, hidden=4096, x="f16", residual=True, out="e4m3"),
        # a prefill chunk of an 8192-wide model
        dict(name="norm_16384x8192_e4m3", op="norm", rows=16384, hidden=8192, x="bf16", residual=True, out="e4m3"),
        # the attention output of a decode batch, ahead of the 8-bit O-projection
        dict(name="quant_64x4096_rows", op="quant", rows=64, cols=4096, x="f16", block_rows=1),
        # one weight matrix laid out in 128 x 128 blocks, ragged at both edges
        dict(name="quant_28672x8200_blocks", op="quant", rows=28672, cols=8200, x="bf16", block_rows=128),
        # one token through a 2048 x 2048 projection, added to the residual stream
        dict(name="linear_1x2048x2048_res", op="linear", m=1, n=2048, k=2048, residual=True, out="f32"),
        # the stacked QKV rows of a 4096-wide model for a decode batch
        dict(name="linear_64x6144x4096", op="linear", m=64, n=6144, k=4096, residual=False, out="f16"),
        # the vocabulary projection of a small odd batch
        dict(name="linear_37x128256x4096", op="linear", m=37, n=128256, k=4096, residual=False, out="f32"),
        # a prefill chunk through the same QKV rows, not a multiple of a tile
        dict(name="linear_8000x6144x4096", op="linear", m=8000, n=6144, k=4096, residual=False, out="bf16"),
        # one sequence, every filter on
        dict(name="sample_1x32000_f32", op="sample", batch=1, vocab=32000, x="f32", filters="all"),
        # a decode batch, each row with settings of its own
        dict(name="sample_64x128256_f32", op="sample", batch=64, vocab=128256, x="f32", filters="mixed"),
        # many sequences over an odd vocabulary, temperature only
        dict(name="sample_256x50257_f16", op="sample", batch=256, vocab=50257, x="f16", filters="none"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "quant", "linear", "linear", "linear", "sample", "sample"])
    if op == "norm":
        hidden = _log(rng, 64, 8192)
        hidden = hidden if rng.random() < 0.3 else max(64, hidden // 64 * 64)
        rows = _log(rng, 1, min(16384, (16384 * 8192) // hidden))
        return dict(op=op, rows=rows, hidden=hidden, x=rng.choice(["f32", "f16", "bf16"]),
                    residual=rng.random() < 0.6, out=rng.choice(["f32", "f16", "bf16", "e4m3", "e4m3"]))
    if op == "quant":
        cols = _log(rng, 64, 8192)
        cols = cols if rng.random() < 0.3 else max(64, cols // 64 * 64)
        block_rows = rng.choice([1, 1, 128])
        return dict(op=op, rows=_log(rng, 1, 16384), cols=cols, x=rng.choice(["f32", "f16", "bf16"]),
                    block_rows=block_rows)
    if op == "linear":
        k = 16 * _log(rng, 8, 512)
        n = _log(rng, 32, 16384)
        n = n if rng.random() < 0.3 else max(32, n // 32 * 32)
        m = _log(rng, 1, 8192)
        while m * n * k > 8000 * 6144 * 4096:
            m = (m + 1) // 2
        return dict(op=op, m=m, n=n, k=k, residual=rng.random() < 0.3, out=rng.choice(["f32", "f16", "bf16"]))
    vocab = _log(rng, 500, 131072)
    return dict(op=op, batch=_log(rng, 1, max(1, min(256, (64 * 128256) // vocab))), vocab=vocab,
                x=rng.choice(["f32", "f16", "bf16"]), filters=rng.choice(["all", "mixed", "mixed", "none"]))


def _groups(n):
    return (n + 127) // 128


def work(case):
    op = case["op"]
    if op == "norm":
        r, h = case["rows"], case["hidden"]
        b = r * h * (SIZE[case["x"]] + (8 if case["residual"] else 0) + SIZE[case["out"]]) + 4 * h
        b += 4 * r * _groups(h) if case["out"] == "e4m3" else 0
        return {"bytes": b, "flops": 6 * r * h}
    if op == "quant":
        r, c = case["rows"], case["cols"]
        s = r * _groups(c) if case["block_rows"] == 1 else _groups(r) * _groups(c)
        return {"bytes": r * c * (SIZE[case["x"]] + 1) + 4 * s, "flops": 3 * r * c}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        g = _groups(k)
        b = m * k + n * k + 4 * g * (m + _groups(n)) + m * n * (SIZE[case["out"]] + (4 if case["residual"] else 0))
        return {"bytes": b, "flops": 2 * m * n * k}
    b, v = case["batch"], case["vocab"]
    return {"bytes": b * v * SIZE[case["x"]] + 28 * b, "flops": 8 * b * v}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _row_scales(y):
    """Per-row scales of groups of 128 columns, [groups][rows]."""
    r, c = y.shape
    g = _groups(c)
    pad = torch.zeros((r, g * 128), dtype=torch.float32, device=y.device)
    pad[:, :c] = y.abs()
    return torch.clamp(pad.view(r, g, 128).amax(-1) / E4M3_MAX, min=TINY).t().contiguous()


def _block_scales(y):
    """Scales of 128 x 128 blocks, [row blocks][column blocks]."""
    r, c = y.shape
    rb, cb = _groups(r), _groups(c)
    pad = torch.zeros((rb * 128, cb * 128), dtype=torch.float32, device=y.device)
    pad[:r, :c] = y.abs()
    return torch.clamp(pad.view(rb, 128, cb, 128).amax(3).amax(1) / E4M3_MAX, min=TINY)


def _spread_rows(s, cols):
    """[groups][rows] scales as one per element, [rows][cols]."""
    return s.t().repeat_interleave(128, dim=1)[:, :cols]


def _spread_blocks(s, rows, cols):
    return s.repeat_interleave(128, dim=0)[:rows].repeat_interleave(128, dim=1)[:, :cols]


def _to_e4m3(y, spread):
    return (y / spread).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)

    def rand(*shape):
        return torch.rand(shape, generator=g, device=DEV, dtype=torch.float32)

    op = case["op"]
    if op == "norm":
        r, h = case["rows"], case["hidden"]
        # a few channels much larger than the rest, as hidden states have them
        channel = 1.0 + 8.0 * (rand(h) > 0.995).float()
        s = {"x": (randn(r, h) * channel).to(DT[case["x"]]), "weight": 1.0 + 0.2 * randn(h), "residual": None}
        if case["residual"]:
            s["residual"] = randn(r, h) * channel * 3.0
            s["stream"] = torch.empty_like(s["residual"])  # the updated stream: the other of a program's two buffers
    elif op == "quant":
        r, c = case["rows"], case["cols"]
        s = {"x": (randn(r, c) * (0.02 if case["block_rows"] == 128 else 1.0)).to(DT[case["x"]])}
    elif op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = randn(m, k)
        xs = _row_scales(x)
        w = randn(n, k) / math.sqrt(k)
        ws = _block_scales(w)
        s = {"x": _to_e4m3(x, _spread_rows(xs, k)), "xs": xs, "w": _to_e4m3(w, _spread_blocks(ws, n, k)), "ws": ws,
             "residual": randn(m, n) if case["residual"] else None}
    else:
        b, v = case["batch"], case["vocab"]
        logits = randn(b, v) * 2.5
        top = (rand(b, 24) * v).long().clamp(max=v - 1)  # a few likely tokens, as a model gives them
        logits.scatter_add_(1, top, 4.0 + 4.0 * rand(b, 24))
        if case["filters"] == "mixed":  # every fourth row under a grammar's mask
            masked = (torch.arange(b, device=DEV) % 4 == 3)[:, None] & (rand(b, v) < 0.7)
            logits.masked_fill_(masked, -math.inf)
        s = {"logits": logits.to(DT[case["x"]]), "u": rand(b), "temperature": 0.6 + 0.8 * rand(b),
             "top_k": None, "top_p": None, "min_p": None}
        if case["filters"] != "none":
            s["top_k"] = 20 + (rand(b) * 180).int()
            s["top_p"] = 0.7 + 0.28 * rand(b)
            s["min_p"] = 0.002 + 0.05 * rand(b)
        if case["filters"] == "mixed":
            kind = (rand(b) * 5).int()  # 0: greedy, 1: top-k only, 2: top-p only, 3: min-p only, 4: all
            s["temperature"] = torch.where(kind == 0, torch.zeros_like(s["temperature"]), s["temperature"])
            off_k = (kind == 2) | (kind == 3)
            s["top_k"] = torch.where(off_k, torch.zeros_like(s["top_k"]), s["top_k"])
            s["top_p"] = torch.where((kind == 1) | (kind == 3), torch.ones_like(s["top_p"]), s["top_p"])
            s["min_p"] = torch.where((kind == 1) | (kind == 2), torch.zeros_like(s["min_p"]), s["min_p"])
    s["case"] = dict(case)
    s["eps"] = 1e-5
    s["out_dtype"] = DT[case["out"]] if "out" in case else None
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _run_norm(s):
    stream = s.get("stream")
    if own:
        got = _lib().rms_norm(s["x"], s["weight"], eps=s["eps"], residual=s["residual"], residual_out=stream,
                              out_dtype=s["out_dtype"])
        y, scales = got if s["out_dtype"] == torch.float8_e4m3fn else (got, None)
        return {"y": y, "scales": scales, "residual": stream}
    h = s["x"].float()
    if s["residual"] is not None:
        h = torch.add(h, s["residual"], out=stream)
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"]
    scales = None
    if s["out_dtype"] == torch.float8_e4m3fn:
        scales = _row_scales(y)
        y = _to_e4m3(y, _spread_rows(scales, y.shape[1]))
    else:
        y = y.to(s["out_dtype"])
    return {"y": y, "scales": scales, "residual": stream}


def _run_quant(s):
    block_rows = s["case"]["block_rows"]
    if own:
        q, scales = _lib().quantize_fp8(s["x"], block_rows=block_rows)
        return {"q": q, "scales": scales}
    x = s["x"].float()
    if block_rows == 1:
        scales = _row_scales(x)
        return {"q": _to_e4m3(x, _spread_rows(scales, x.shape[1])), "scales": scales}
    scales = _block_scales(x)
    return {"q": _to_e4m3(x, _spread_blocks(scales, *x.shape)), "scales": scales}


def _run_linear(s):
    if own:
        return _lib().fp8_linear(s["x"], s["xs"], s["w"], s["ws"], residual=s["residual"], out_dtype=s["out_dtype"])
    (m, k), n = s["x"].shape, s["w"].shape[0]
    x = s["x"].float() * _spread_rows(s["xs"], k)
    w = s["w"].float() * _spread_blocks(s["ws"], n, k)
    y = x @ w.t()
    if s["residual"] is not None:
        y = y + s["residual"]
    return y.to(s["out_dtype"])


def _run_sample(s):
    if own:
        tokens, logprobs = _lib().sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                                top_p=s["top_p"], min_p=s["min_p"], return_logprobs=True)
        return {"tokens": tokens, "logprobs": logprobs}
    # 64 bits: a token is chosen where a long sum passes a border
    x = s["logits"].double()
    b, v = x.shape
    order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: lowest index first
    z, idx = order.values, order.indices
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()
    w = torch.exp((z - z[:, :1]) / t[:, None])
    rank = torch.arange(v, device=x.device)
    keep = w > 0
    if s["top_k"] is not None:
        k = torch.where((s["top_k"] <= 0) | (s["top_k"] > v), torch.full_like(s["top_k"], v), s["top_k"])
        keep = keep & (rank[None, :] < k[:, None])
    w = torch.where(keep, w, torch.zeros_like(w))
    if s["top_p"] is not None:
        cum = w.cumsum(1)
        p = s["top_p"].double()
        before = cum - w  # kept while what stands before falls short of the share
        keep = keep & ((p >= 1.0)[:, None] | (before < p[:, None] * cum[:, -1:]) | (rank == 0))
    if s["min_p"] is not None:
        keep = keep & ((w >= s["min_p"].double()[:, None]) | (rank == 0))
    keep = torch.where(greedy[:, None], rank[None, :] == 0, keep)
    w = torch.where(keep, w, torch.zeros_like(w))
    by_index = torch.zeros_like(w).scatter_(1, idx, w)
    cum = by_index.cumsum(1)
    total = cum[:, -1:]
    tokens = (cum > s["u"].double()[:, None] * total).to(torch.uint8).argmax(1)
    logprobs = torch.log(by_index.gather(1, tokens[:, None]) / total)[:, 0]
    return {"tokens": tokens.to(torch.int32), "logprobs": logprobs.float()}


def run(state):
    return {"norm": _run_norm, "quant": _run_quant, "linear": _run_linear, "sample": _run_sample}[state["case"]["op"]](
        state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits (an e4m3 output stands for the value before its
# rounding, in units of its scale)
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        rows, hidden = case["rows"], case["hidden"]
        h = s["x"].to(torch.float64)
        if s["residual"] is not None:
            h += s["residual"]
        stream = h.clone() if s["residual"] is not None else None
        h *= (1.0 / torch.sqrt((h * h).sum(1) / hidden + s["eps"]))[:, None]
        h *= s["weight"].double()[None, :]
        if case["out"] != "e4m3":
            return {"y": h, "scales": None, "residual": stream}
        scales = torch.empty((_groups(hidden), rows), dtype=torch.float64, device=DEV)
        for j in range(_groups(hidden)):
            part = h[:, j * 128:(j + 1) * 128]
            scales[j] = torch.clamp(part.abs().amax(1) / E4M3_MAX, min=TINY)
            part /= scales[j][:, None]
        return {"y": h, "scales": scales, "residual": stream}
    if op == "quant":
        x = s["x"].to(torch.float64)
        rows, cols = x.shape
        rb = case["block_rows"]
        scales = torch.empty((_groups(cols), rows) if rb == 1 else (_groups(rows), _groups(cols)),
                             dtype=torch.float64, device=DEV)
        for j in range(_groups(cols)):
            part = x[:, j * 128:(j + 1) * 128]
            top = part.abs().amax(1)
            if rb == 1:
                scales[j] = torch.clamp(top / E4M3_MAX, min=TINY)
                part /= scales[j][:, None]
                continue
            full = torch.zeros(_groups(rows) * 128, dtype=torch.float64, device=DEV)
            full[:rows] = top
            scales[:, j] = torch.clamp(full.view(-1, 128).amax(1) / E4M3_MAX, min=TINY)
            part /= scales[:, j].repeat_interleave(128)[:rows][:, None]
        return {"q": x, "scales": scales}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros((m, n), dtype=torch.float64, device=DEV)
        for j in range(_groups(k)):
            a = s["x"][:, j * 128:(j + 1) * 128].double() * s["xs"][j].double()[:, None]
            b = s["w"][:, j * 128:(j + 1) * 128].double()
            b *= s["ws"][:, j].double().repeat_interleave(128)[:n][:, None]
            y.addmm_(a, b.t())
        if s["residual"] is not None:
            y += s["residual"]
        return y
    # sampling, one row at a time, by a walk over the sorted order
    logits = s["logits"].double()
    b, v = logits.shape
    tokens, logprobs = [], []
    value = {n: (s[n].tolist() if s[n] is not None else [d] * b)
             for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    u = s["u"].tolist()
    for r in range(b):
        t = value["temperature"][r]
        top, first = logits[r].max(0)
        if t <= 0:
            tokens.append(int((logits[r] == top).nonzero()[0, 0]))
            logprobs.append(0.0)
            continue
        z, at = logits[r].sort(descending=True, stable=True)
        n = int((z > -math.inf).sum())
        k = value["top_k"][r]
        n = min(n, k) if 0 < k else n
        w = ((z[:n] - top) / t).exp()
        sums = w.cumsum(0)
        if value["top_p"][r] < 1.0:
            n = min(n, int((sums < value["top_p"][r] * sums[-1]).sum()) + 1)
        n = min(n, max(1, int((w >= value["min_p"][r]).sum())))
        kept, by = at[:n].sort()
        w = w[:n][by]
        sums = w.cumsum(0)
        i = min(n - 1, int((sums <= u[r] * sums[-1]).sum()))
        tokens.append(int(kept[i]))
        logprobs.append(math.log(float(w[i]) / float(sums[-1])))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
