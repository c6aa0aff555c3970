"""Token sampling against a walk over the sorted candidates in 64 bits.

Tokens have to be equal, except where the draw lies within 1e-9 of a border (the
fixed-point weights are off by 2^-44 of the largest each, at most 2^18 of them).
The log-probability is one fp32 rounding (2^-24 of it) from a value that the
weights' rounding leaves within 1e-8.
"""
import numpy as np
import pytest
import torch

import lowp_ref as ref

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"
INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _dev(v, dtype):
    return None if v is None else torch.as_tensor(v, dtype=dtype).to(DEV)


def _run(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    tok, lp = cb.sample_tokens(logits.to(DEV), _dev(u, torch.float32), temperature=_dev(temperature, torch.float32),
                               top_k=_dev(top_k, torch.int32), top_p=_dev(top_p, torch.float32),
                               min_p=_dev(min_p, torch.float32), return_logprobs=True, status=st)
    torch.cuda.synchronize()
    return tok.cpu(), lp.cpu(), int(st.item())


def _check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    tok, lp, status = _run(logits, u, temperature, top_k, top_p, min_p)
    x = logits.float().numpy()
    empty = False
    for b in range(len(x)):
        pick = lambda v, d: d if v is None else float(np.float32(v[b]))  # noqa: E731
        want, wlp, _ = ref.sample(x[b], pick(u, 0), pick(temperature, 1.0), int(pick(top_k, 0)), pick(top_p, 1.0),
                                  pick(min_p, 0.0))
        if want is None:
            continue
        empty |= want == -1
        assert int(tok[b]) == want, b
        if want >= 0:
            assert abs(float(lp[b]) - wlp) <= abs(wlp) * 2.0 ** -24 + 2e-8, b
        else:
            assert float(lp[b]) == -INF
    assert status == (cb.STATUS_NO_TOKEN if empty else 0)


def _logits(batch, vocab, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(batch, vocab, generator=g) * scale).to(dtype), torch.rand(batch, generator=g)


VOCABS = [1, 2, 31, 100, 513, 1000, 4099, 32000, 50257]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_temperature_only(vocab, dtype):
    x, u = _logits(5, vocab, dtype, vocab)
    _check(x, u)
    _check(x, u, temperature=[0.3, 0.9, 1.0, 1.7, 5.0])


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_each_filter(vocab, dtype):
    x, u = _logits(6, vocab, dtype, vocab + 1)
    _check(x, u, top_k=[1, 2, 7, 50, 3000, vocab])
    _check(x, u, top_p=[0.01, 0.3, 0.6, 0.9, 0.97, 0.999])
    _check(x, u, min_p=[1.0, 0.5, 0.1, 0.01, 1e-4, 1e-20])
    _check(x, u, temperature=[0.5, 0.7, 1.0, 1.0, 1.3, 2.0], top_k=[1, 5, 40, 200, 1000, 20000],
           top_p=[0.9, 0.5, 0.9, 0.95, 0.8, 0.99], min_p=[0.0, 0.0, 0.02, 0.01, 0.1, 0.001])


@pytest.mark.parametrize("batch", [1, 3, 19, 80, 300])
def test_batches(batch):
    """Every cluster size: one row to more rows than SMs."""
    vocab = 40000 if batch < 20 else 9001
    x, u = _logits(batch, vocab, torch.float32, batch)
    if batch > 100:  # (the walk in Python is slow: a few of the rows)
        tok, _, _ = _run(x, u, top_k=[30] * batch, top_p=[0.9] * batch)
        for b in range(0, batch, 29):
            want, _, _ = ref.sample(x[b].numpy(), float(u[b]), 1.0, 30, float(np.float32(0.9)))
            assert want is None or int(tok[b]) == want
        return
    _check(x, u, top_k=[30] * batch, top_p=[0.9] * batch)


def test_flat_rows_and_ties():
    """Equal logits: order by index alone; more members of a bin than the list holds; wide nuclei."""
    v = 30011
    x = torch.zeros(7, v)
    x[1] = -3.4028234663852886e38            # every logit the type's lowest
    x[2, ::2] = 1.0                           # two levels
    x[3] = torch.linspace(0, 1e-3, v)         # all of one level-one bin, distinct
    x[4] = torch.randn(v, generator=torch.Generator().manual_seed(4)) * 0.01
    x[5, :20000] = -0.0                       # -0 and +0 are one value
    x[6] = (torch.arange(v) % 7).float() * 0.125
    u = torch.tensor([0.37, 0.999, 0.5, 0.25, 0.75, 0.6, 0.9])
    _check(x, u)
    _check(x, u, top_k=[12345, 9000, 20000, 5000, 25000, 20001, 3])
    _check(x, u, top_p=[0.5, 0.123, 0.9, 0.3, 0.6, 0.7, 0.05])
    _check(x, u, top_k=[12345, 9000, 20000, 5000, 25000, 20001, 3000], top_p=[0.5, 0.123, 0.9, 0.3, 0.6, 0.7, 0.05])


def test_masks_infinities_and_nan():
    v = 2051
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, v, generator=g)
    x[0] = -INF                               # nothing left
    x[1] = float("nan")
    x[2] = -INF
    x[2, 777] = -5.0                          # one left
    x[3, torch.rand(v, generator=g) < 0.9] = -INF   # fewer left than top_k
    x[4, torch.rand(v, generator=g) < 0.5] = float("nan")
    x[5, 100] = x[5, 900] = INF               # the infinities share the draw
    x[6] = -3.4028234663852886e38             # masked with the type's lowest value
    x[6, 5:9] = 1.0
    x[7, :1000] = 3.4028234663852886e38       # distances past fp32
    x[7, 1000:] = -3.4028234663852886e38
    u = torch.rand(9, generator=g)
    for kw in (dict(), dict(top_k=[300] * 9), dict(top_p=[0.9] * 9), dict(min_p=[0.05] * 9),
               dict(temperature=[0.0] * 9), dict(temperature=[0.7] * 9, top_k=[500] * 9, top_p=[0.95] * 9, min_p=[0.001] * 9)):
        _check(x, u, **kw)
    assert torch.equal(_run(x, u, temperature=[0.0] * 9)[0][:2], torch.tensor([-1, -1], dtype=torch.int32))


def test_settings_out_of_range():
    x, _ = _logits(8, 500, torch.float32, 77)
    u = torch.tensor([-1.0, 0.0, 1.0, 2.0, float("nan"), 0.99999994, 0.5, 0.5])
    nan = float("nan")
    tok, lp, _ = _run(x, u)
    assert torch.isfinite(lp).all() and torch.all((tok >= 0) & (tok < 500))
    assert int(tok[0]) == int(tok[1].new_tensor(ref.sample(x[0].numpy(), 0.0)[0]))
    assert int(tok[4]) == ref.sample(x[4].numpy(), 0.0)[0]
    half = [0.5] * 8
    off = _run(x, half)[0]
    assert torch.equal(_run(x, half, top_k=[0, -1, 500, 501, 2 ** 31 - 1, -2 ** 31, 0, 0])[0], off)
    assert torch.equal(_run(x, half, top_p=[1.0, 1.5, nan, INF, 1.0, 1.0, 1.0, 1.0])[0], off)
    assert torch.equal(_run(x, half, min_p=[0.0, -1.0, nan, -INF, 0.0, 0.0, 0.0, 0.0])[0], off)
    first = x.argmax(1).int()
    for kw in (dict(temperature=[0.0, -1.0, nan, -INF] * 2), dict(top_k=[1] * 8), dict(top_p=[0.0, -1.0, -INF, 1e-9] * 2),
               dict(min_p=[1.0, 1.5, INF, 2.0] * 2), dict(temperature=[1e-45] * 8)):
        tok, lp, _ = _run(x, half, **kw)
        assert torch.equal(tok, first) and torch.all(lp == 0)
    _check(x, half, temperature=[1e30] * 8)  # flat


def test_shares_follow_the_weights():
    """4096 evenly spaced draws of one row: each token's share is its probability to one draw in 4096, twice."""
    n = 4096
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, -INF, 0.5]).repeat(n, 1)
    tok, _, _ = _run(x, (torch.arange(n) + 0.5) / n)
    share = torch.bincount(tok, minlength=6) / n
    assert torch.all((share - torch.softmax(x[0], 0)).abs() <= 2 / n)
    assert torch.all(tok[1:] >= tok[:-1])


def test_largest_vocabulary():
    v = 327680
    x, u = _logits(2, v, torch.float32, 8)
    tok, lp, _ = _run(x, u, top_k=[100, 0], top_p=[1.0, 0.5])
    for b, kw in ((0, dict(top_k=100)), (1, dict(top_p=0.5))):
        want, wlp, _ = ref.sample(x[b].numpy(), float(u[b]), **kw)
        if want is not None:
            assert int(tok[b]) == want and abs(float(lp[b]) - wlp) <= abs(wlp) * 2.0 ** -24 + 2e-8


def test_logits_past_32_bits():
    """More than 2^31 logits: the last rows' tokens equal those of a call of their own, filter by filter."""
    batch, vocab, last = 17000, 128256, 160
    logits = torch.empty(batch, vocab, dtype=torch.float16, device=DEV)
    logits[:500].normal_()
    logits[500:] = logits[:500].repeat(33, 1)
    logits[-last:].normal_()
    assert logits.numel() > 1 << 31
    u = torch.rand(batch, device=DEV)
    p, k = torch.full((batch,), 0.7, device=DEV), torch.full((batch,), 30, dtype=torch.int32, device=DEV)
    for kw in (dict(), dict(top_p=p), dict(top_k=k, top_p=p)):
        got = cb.sample_tokens(logits, u, **kw)
        part = cb.sample_tokens(logits[-last:], u[-last:], **{n: t[-last:] for n, t in kw.items()})
        assert torch.equal(got[-last:], part)


def test_writes_its_rows_only_and_refuses():
    x, u = _logits(3, 100, torch.float32, 1)
    x, u = x.to(DEV), u.to(DEV)
    out = torch.full((5,), 77, dtype=torch.int32, device=DEV)
    cb.sample_tokens(x, u, out=out[1:4])
    assert out[0] == 77 and out[4] == 77 and torch.all(out[1:4] < 100)
    assert torch.equal(cb.sample_tokens(x, u), out[1:4])
    with pytest.raises(ValueError, match="uniforms"):
        cb.sample_tokens(x, u[:2])
    with pytest.raises(TypeError):
        cb.sample_tokens(x, u, top_k=u)
    with pytest.raises(ValueError, match="contiguous"):
        cb.sample_tokens(x[:, ::2], u)
    with pytest.raises(cb.CottusError) as e:
        cb.sample_tokens(torch.zeros(1, 327681, device=DEV), u[:1])
    assert e.value.code == cb.COTTUS_ERR_UNSUPPORTED
    assert cb.sample_tokens(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("batch", [1, 64, 320])
def test_top_p_alone(batch):
    """Rows on which a count of the distances says much, little or something wrong about where the mass ends: smooth,
    peaked, sorted (one part of the row holds every likely token), crowded just below the maximum, in a few steps, at
    steep and flat temperatures, with shares of nearly nothing and nearly everything."""
    vocab = 30011
    g = torch.Generator().manual_seed(21)
    rows = [torch.randn(vocab, generator=g) * s for s in (0.02, 1.0, 4.0)]
    rows.append(torch.randn(vocab, generator=g).sort(descending=True).values * 2)
    peaked = torch.randn(vocab, generator=g)
    peaked[torch.randint(vocab, (30,), generator=g)] += 9 + torch.rand(30, generator=g)
    rows.append(peaked)
    crowded = torch.randn(vocab, generator=g) - 6
    crowded[::20] = 4.0 + 0.02 * torch.rand(crowded[::20].numel(), generator=g)
    crowded[77] = 4.25
    rows += [crowded, (torch.randn(vocab, generator=g) * 2).round(), torch.linspace(-30, 5, vocab)]
    n = len(rows)
    shares, temps = (1e-6, 0.1, 0.5, 0.9, 0.99, 0.999999), (0.05, 0.7, 1.0, 30.0)
    cases = [(i % n, float(np.float32(shares[(i // 3) % 6])), float(np.float32(temps[i % 4]))) for i in range(batch)]
    logits = torch.stack([rows[r] for r, _, _ in cases])
    u = torch.rand(batch, generator=g)
    p, t = torch.tensor([c[1] for c in cases]), torch.tensor([c[2] for c in cases])
    got = cb.sample_tokens(logits.to(DEV), u.to(DEV), temperature=t.to(DEV), top_p=p.to(DEV))
    again = cb.sample_tokens(logits.to(DEV), u.to(DEV), temperature=t.to(DEV), top_p=p.to(DEV))
    assert torch.equal(got, again)
    known = 0
    for b in range(0, batch, max(1, batch // 96)):
        want, _, _ = ref.sample(logits[b].numpy(), float(u[b]), cases[b][2], 0, cases[b][1])
        if want is None:
            continue
        known += 1
        assert int(got[b]) == want, (b, cases[b])
    assert known >= min(batch, 96) * 0.8
