"""64-bit definitions of the norm, 8-bit and sampling operators for the tests
(numpy / torch on the CPU, written from the formulas)."""
import numpy as np
import torch

E4M3_MAX, TINY = 448.0, 2.0 ** -126


def groups(n):
    return (n + 127) // 128


def row_scales(y):
    """[groups][rows] fp32 scales of fp32 y, by the fp32 formula."""
    r, c = y.shape
    pad = torch.zeros(r, groups(c) * 128, dtype=torch.float32)
    pad[:, :c] = y.abs()
    return torch.clamp(pad.view(r, -1, 128).amax(-1) / E4M3_MAX, min=TINY).t().contiguous()


def block_scales(y):
    r, c = y.shape
    pad = torch.zeros(groups(r) * 128, groups(c) * 128, dtype=torch.float32)
    pad[:r, :c] = y.abs()
    return torch.clamp(pad.view(groups(r), 128, groups(c), 128).amax(3).amax(1) / E4M3_MAX, min=TINY)


def spread_rows(s, cols):
    return s.t().repeat_interleave(128, 1)[:, :cols]


def spread_blocks(s, rows, cols):
    return s.repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def to_e4m3(y, spread):
    return (y / spread).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def dequant_rows(q, s):
    return q.double() * spread_rows(s.double(), q.shape[1])


def dequant_blocks(q, s):
    return q.double() * spread_blocks(s.double(), *q.shape)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability, kept indices) of one row: the definition, walked
    in Python over the sorted candidates.  The draw `u` may come back as None
    where it lies within 1e-9 of a border (no token is asserted then)."""
    x = np.asarray(logits, np.float64)
    cand = [i for i in range(len(x)) if x[i] > -np.inf]
    if not cand:
        return -1, -np.inf, []
    cand.sort(key=lambda i: (-x[i], i))
    if not temperature > 0:
        return cand[0], 0.0, cand[:1]
    top = x[cand[0]]

    def weight(i):
        if x[i] == top:
            return 1.0
        return 0.0 if np.isinf(top) else float(np.exp((x[i] - top) / temperature))

    w = {i: weight(i) for i in cand}
    kept = cand[:top_k] if 0 < top_k < len(cand) else cand
    if top_p < 1.0:
        target, run, n = top_p * sum(w[i] for i in kept), 0.0, 0
        while n < len(kept):
            run += w[kept[n]]
            n += 1
            if run >= target:
                break
        kept = kept[:n]
    if min_p > 0:
        kept = kept[:1] + [i for i in kept[1:] if w[i] >= min_p]
    total = sum(w[i] for i in kept)
    run, t = 0.0, min(max(u, 0.0), 1.0 - 2.0 ** -24) * total
    for i in sorted(kept):
        run += w[i]
        if abs(run - t) < 1e-9 * total and w[i] < total and t > 0:
            return None, None, kept
        if run > t:
            return i, float(np.log(w[i] / total)), kept
    raise AssertionError("the running sum ends at the total")
