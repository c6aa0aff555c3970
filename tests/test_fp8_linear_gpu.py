"""The block-scaled e4m3 product against its definition in 64 bits.

A product of two e4m3 values is exact in fp32.  Bound: the tensor core adds at
most 128 products of a group in fp32, each addition off by a step at most
(2^-23 of the largest magnitude on the way, which the sum of magnitudes
bounds); the groups' sums take one fused multiply-add each, the scales' product
one rounding, the splits at most 8 additions and the residual one; then the
output is rounded once.
"""
import pytest
import torch

import lowp_ref as ref

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"
FP8 = torch.float8_e4m3fn
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def _quantised(m, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))
    w = torch.randn(n, k, generator=g) / k ** 0.5
    xs, ws = ref.row_scales(x), ref.block_scales(w)
    return ref.to_e4m3(x, ref.spread_rows(xs, k)), xs, ref.to_e4m3(w, ref.spread_blocks(ws, n, k)), ws


def _check(got, x, xs, w, ws, res):
    a, b = ref.dequant_rows(x, xs), ref.dequant_blocks(w, ws)
    y, mag = a @ b.t(), a.abs() @ b.abs().t()
    if res is not None:
        y, mag = y + res.double(), mag + res.abs().double()
    tol = mag * (128 + ref.groups(x.shape[1]) + 11) * 2.0 ** -23 + y.abs() * HALF[got.dtype] + \
        (2.0 ** -25 if got.dtype == torch.float16 else 0)
    assert torch.all((got.cpu().double() - y).abs() <= tol)


# (m, n, k): one row; ragged everything; one group and part of one; several row
# tiles; tiles enough for the wide kernel, with ragged edges in m and n
SHAPES = [(1, 128, 128), (1, 1, 16), (3, 5, 48), (8, 128, 256), (16, 256, 2048), (37, 1000, 1104), (64, 130, 4096),
          (100, 640, 144), (127, 257, 272), (128, 384, 512), (129, 512, 384), (200, 96, 2064), (300, 1001, 528),
          (1300, 3800, 144), (2500, 2050, 272)]


@pytest.mark.parametrize("m, n, k", SHAPES)
def test_small_integers_are_exact(m, n, k):
    """Integers up to 8 with scales that are powers of two: every sum is exact in fp32, so the result has to be."""
    g = torch.Generator().manual_seed(m + n + k)
    x = torch.randint(-8, 9, (m, k), generator=g).float()
    w = torch.randint(-8, 9, (n, k), generator=g).float()
    xs = 2.0 ** torch.randint(-2, 3, (ref.groups(k), m), generator=g)
    ws = 2.0 ** torch.randint(-2, 3, (ref.groups(n), ref.groups(k)), generator=g)
    st = _status()
    got = cb.fp8_linear(x.to(FP8).to(DEV), xs.to(DEV), w.to(FP8).to(DEV), ws.to(DEV), out_dtype=torch.float32, status=st)
    want = (ref.dequant_rows(x, xs).to(DEV) @ ref.dequant_blocks(w, ws).to(DEV).t()).float()
    assert int(st.item()) == 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("out_dtype, residual", [(torch.float32, False), (torch.float16, True), (torch.bfloat16, False),
                                                 (torch.float32, True)])
def test_against_64_bits(m, n, k, out_dtype, residual):
    x, xs, w, ws = _quantised(m, n, k, m * 31 + n * 7 + k)
    res = torch.randn(m, n) if residual else None
    st = _status()
    got = cb.fp8_linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), residual=None if res is None else res.to(DEV),
                        out_dtype=out_dtype, status=st)
    assert got.dtype == out_dtype and int(st.item()) == 0
    _check(got, x, xs, w, ws, res)


# around the borders between the tiles: rows of x, a ring shorter than the groups of one CTA, every number of splits,
# the wide tile with rows that its stores cannot take whole
BORDERS = [(m, n, k) for m in (2, 15, 17, 31, 32, 33, 63, 65, 96) for n, k in ((260, 1040), (20001, 2064))] + \
    [(16, 128 * t, 1152) for t in (1, 13, 18, 22, 29, 37, 49, 73, 74, 100, 148, 149)] + \
    [(17, 128 * t, 1152) for t in (1, 13, 18)] + [(900, 3001, 400), (513, 9000, 16), (257, 10001, 128)] + \
    [(m, n, k) for m in (1, 7, 8, 9, 16) for n, k in ((16, 16), (17, 2048), (2368, 4096), (2369, 4112), (9472, 1040), (9489, 144),
                                                     (130, 8192), (130, 8208))]


@pytest.mark.parametrize("m, n, k", BORDERS)
def test_tile_borders(m, n, k):
    x, xs, w, ws = _quantised(m, n, k, m + n + k)
    res = torch.randn(m, n, generator=torch.Generator().manual_seed(n))
    dev = [t.to(DEV) for t in (x, xs, w, ws)]
    _check(cb.fp8_linear(*dev), x, xs, w, ws, None)
    _check(cb.fp8_linear(*dev, residual=res.to(DEV), out_dtype=torch.float32), x, xs, w, ws, res)


def test_elements_past_32_bits():
    """More than 2^31 results: the last rows equal those of a call of their own (the same tiles)."""
    m, n, k, last = 40000, 56000, 128, 2000
    g = torch.Generator(device=DEV).manual_seed(12)
    x, xs = cb.quantize_fp8(torch.randn(m, k, generator=g, device=DEV))
    w, ws = cb.quantize_fp8(torch.randn(n, k, generator=g, device=DEV), block_rows=128)
    y = cb.fp8_linear(x, xs, w, ws)
    tail = cb.fp8_linear(x[-last:], xs[:, -last:].contiguous(), w, ws)
    assert y.numel() > 1 << 31 and torch.equal(y[-last:], tail)
    head = cb.fp8_linear(x[:last], xs[:, :last].contiguous(), w, ws)
    assert torch.equal(y[:last], head)


def test_long_sums_keep_32_bits():
    """Products of 2^16 and of 2^-6 in one group: the sum needs 23 bits, so a narrower accumulator shows."""
    x = torch.full((4, 128), 2.0 ** -3)
    w = torch.full((128, 128), 2.0 ** -3)
    x[:, 0] = w[:, 0] = 256.0
    one = torch.ones(1, 4), torch.ones(1, 1)
    got = cb.fp8_linear(x.to(FP8).to(DEV), one[0].to(DEV), w.to(FP8).to(DEV), one[1].to(DEV), out_dtype=torch.float32)
    assert torch.all(got == 65536.0 + 127 * 2.0 ** -6)


def test_residual_in_place_and_determinism():
    x, xs, w, ws = _quantised(50, 1024, 2048, 5)
    args = [t.to(DEV) for t in (x, xs, w, ws)]
    res = torch.randn(50, 1024, device=DEV)
    a = cb.fp8_linear(*args, residual=res, out_dtype=torch.float32)
    stream = res.clone()
    b = cb.fp8_linear(*args, residual=stream, out=stream)
    assert b.data_ptr() == stream.data_ptr() and torch.equal(a, b)
    for _ in range(5):
        assert torch.equal(a, cb.fp8_linear(*args, residual=res, out_dtype=torch.float32))
    # weight rows of a whole matrix, cut at its scale blocks
    part = cb.fp8_linear(args[0], args[1], args[2][256:512], args[3][2:4], residual=res[:, 256:512].contiguous(),
                         out_dtype=torch.float32)
    whole = cb.fp8_linear(*args, residual=res, out_dtype=torch.float32)[:, 256:512]
    assert torch.allclose(part, whole, rtol=1e-5, atol=1e-4)  # (another number of splits: the order of the sums differs)


def test_writes_its_rows_only():
    x, xs, w, ws = _quantised(5, 130, 256, 9)
    for dtype in (torch.float32, torch.float16):
        buf = torch.full((7, 130), 7.0, dtype=dtype, device=DEV)
        cb.fp8_linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), out=buf[1:6])
        _check(buf[1:6], x, xs, w, ws, None)
        assert torch.all(buf[0] == 7) and torch.all(buf[6] == 7)


def test_nan_stays_in_its_row_and_column():
    x, xs, w, ws = _quantised(20, 300, 384, 11)
    xs[1, 7] = float("nan")
    x.view(torch.uint8)[3, 200] = 0x7F
    w.view(torch.uint8)[260, 17] = 0x7F
    got = cb.fp8_linear(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), out_dtype=torch.float32).cpu()
    nan = torch.zeros(20, 300, dtype=torch.bool)
    nan[7] = nan[3] = True
    nan[:, 260] = True
    assert torch.equal(torch.isnan(got), nan)


def test_refusals():
    x, xs, w, ws = (t.to(DEV) for t in _quantised(4, 256, 256, 1))
    with pytest.raises(cb.CottusError) as e:
        cb.fp8_linear(x[:, :24].contiguous(), xs[:1].contiguous(), w[:, :24].contiguous(), ws[:, :1].contiguous())
    assert e.value.code == cb.COTTUS_ERR_UNSUPPORTED
    with pytest.raises(TypeError):
        cb.fp8_linear(x.float(), xs, w, ws)
    with pytest.raises(ValueError, match="x_scales"):
        cb.fp8_linear(x, xs.t().contiguous(), w, ws)
    with pytest.raises(ValueError, match="weight_scales"):
        cb.fp8_linear(x, xs, w, ws[:1])
    with pytest.raises(ValueError, match="weight"):
        cb.fp8_linear(x, xs, w[:, :128].contiguous(), ws)
    with pytest.raises(cb.CottusError, match="overlaps"):
        res = torch.zeros(4, 256, device=DEV)
        cb.fp8_linear(x, xs, w, ws, residual=res, out=res.view(-1).view(torch.float16)[:1024].view(4, 256))
    assert cb.fp8_linear(x[:0], xs[:, :0], w, ws).shape == (0, 256)
