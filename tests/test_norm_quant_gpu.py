"""RMS norm (with the residual's addition and the e4m3 output) and e4m3
quantisation against their definitions in 64 bits.

Bounds, in u = 2^-24 (half an fp32 step): the sum of squares adds positive
terms, at most max(32, hidden / 512) + 10 of them in a row in one thread and
over the block, so it is off by that many u; the root halves that; division by
the width, the addition of eps, the root and the two products add a step each
(6).  An output of 16 bits is then rounded once (half a step, 2^-25 absolute
among fp16's subnormals).  An e4m3 value is off by half a step: 2^-4 of it, or
2^-10 of its scale among the subnormals.
"""
import pytest
import torch

import lowp_ref as ref

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _inputs(rows, hidden, dtype, residual, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 7 + hidden)
    x = torch.randn(rows, hidden, generator=g).to(dtype)
    x[:, 0] *= 20
    w = 1.0 + 0.3 * torch.randn(hidden, generator=g)
    r = 3 * torch.randn(rows, hidden, generator=g) if residual else None
    return x, w, r


def _expected(x, w, r, eps):
    h = x.float() if r is None else x.float() + r
    y = h.double()
    y = y / torch.sqrt(y.square().mean(1, keepdim=True) + eps) * w.double()
    rel = ((max(32, x.shape[1] / 512) + 10) / 2 + 6) * U
    return h, y, rel


def _check_y(y, got, rel):
    tol = y.abs() * (rel + HALF[got.dtype] * (1 + rel)) + TINY[got.dtype]
    assert torch.all((got.cpu().double() - y).abs() <= tol)


def _check_e4m3(y, q, s, rel):
    q, s = q.cpu(), s.cpu()
    ys = ref.row_scales(y.float())  # (the fp32 rounding of y is one u)
    assert torch.all((s.double() - ys.double()).abs() <= ys.double() * (rel + 3 * U))
    spread = ref.spread_rows(s.double(), y.shape[1])
    tol = torch.maximum(y.abs() * 2.0 ** -4, spread * 2.0 ** -10) * (1 + 2.0 ** -10) + y.abs() * rel
    assert torch.all((q.double() * spread - y).abs() <= tol)


# one row to several waves; whole groups, ragged groups, odd widths, widths
# around the register kernel's limits (8 * 1024, 8 * 2048, 8 * 4096) and past them
SHAPES = [(1, 2048), (3, 128), (5, 8), (2, 136), (7, 1), (4, 127), (3, 129), (6, 4096), (2, 4104), (2, 8192), (2, 8200),
          (1, 32768), (1, 32776), (1000, 264), (33, 4999)] + \
    [(70, 2047), (5, 2049), (4, 8191), (2, 8195), (3, 16383), (2, 16385), (1, 32767)] + \
    [(149, 1032), (300, 8200), (150, 16384), (2, 16392), (1300, 136), (1200, 4104)]  # and by rows per SM


@pytest.mark.parametrize("rows, hidden", SHAPES)
@pytest.mark.parametrize("x_dtype, out_dtype, residual", [
    (torch.float32, torch.float16, False), (torch.float16, FP8, True), (torch.bfloat16, FP8, False),
    (torch.float32, torch.float32, True), (torch.bfloat16, torch.bfloat16, True), (torch.float16, torch.float32, False),
])
def test_rms_norm(rows, hidden, x_dtype, out_dtype, residual):
    x, w, r = _inputs(rows, hidden, x_dtype, residual)
    h, y, rel = _expected(x, w, r, 1e-5)
    rd = r.to(DEV) if residual else None
    got = cb.rms_norm(x.to(DEV), w.to(DEV), eps=1e-5, residual=rd, out_dtype=out_dtype)
    torch.cuda.synchronize()
    if residual:  # one fp32 addition, in place
        assert torch.equal(rd.cpu(), h)
    if out_dtype == FP8:
        _check_e4m3(y, *got, rel)
    else:
        assert got.dtype == out_dtype
        _check_y(y, got, rel)


@pytest.mark.parametrize("hidden", [136, 1032, 4096, 8192, 8200, 12288, 16384, 32768])
@pytest.mark.parametrize("x_dtype, residual", [(torch.float16, False), (torch.float32, True)])
def test_rows_do_not_depend_on_their_number(hidden, x_dtype, residual):
    """A row of a batch equals, bit for bit, the same row alone (the kernel's split of a row over threads differs)."""
    x, w, r = (None if t is None else t.to(DEV) for t in _inputs(1300, hidden, x_dtype, residual))
    for out_dtype in (torch.float32, FP8):
        def norm(k):
            got = cb.rms_norm(x[:k], w, residual=None if r is None else r[:k].clone(), out_dtype=out_dtype)
            return (got[0].float(), got[1]) if out_dtype == FP8 else (got,)
        full = norm(1300)
        for k in (1, 140, 200):
            part = norm(k)
            assert torch.equal(part[0], full[0][:k])
            if out_dtype == FP8:
                assert torch.equal(part[1], full[1][:, :k])


def test_rms_norm_buffers_and_aliases():
    x, w, r = _inputs(9, 512, torch.float32, True)
    h, y, rel = _expected(x, w, r, 1e-6)
    xd, wd, rd = x.to(DEV), w.to(DEV), r.to(DEV)
    # the stream into another buffer: the residual stays
    ro = torch.full_like(rd, float("nan"))
    a = cb.rms_norm(xd, wd, eps=1e-6, residual=rd, residual_out=ro)
    assert torch.equal(ro.cpu(), h) and torch.equal(rd.cpu(), r)
    _check_y(y, a, rel)
    # the output over the input (fp32, and an odd width through the other kernel)
    b = cb.rms_norm(xd, wd, eps=1e-6, residual=rd, residual_out=ro, out=xd)
    assert b.data_ptr() == xd.data_ptr() and torch.equal(a, b)
    x, w, _ = _inputs(9, 333, torch.float16, False)
    xd, wd = x.to(DEV), w.to(DEV)
    a = cb.rms_norm(xd, wd)
    b = cb.rms_norm(xd, wd, out=xd)
    assert torch.equal(a, b)
    # rows that start off a 16-byte boundary
    big = torch.zeros(9 * 512 + 1, dtype=torch.float16, device=DEV)
    off = big[1:].view(9, 512)
    off.copy_(torch.randn(9, 512))
    w = torch.ones(512, device=DEV)
    assert torch.allclose(cb.rms_norm(off, w).float(), cb.rms_norm(off.clone(), w).float(), rtol=2.0 ** -10, atol=0)
    assert big[0] == 0


@pytest.mark.parametrize("hidden", [256, 250])
def test_rms_norm_special_rows(hidden):
    x = torch.randn(5, hidden)
    x[0] = 0                     # eps alone: zeros
    x[1, 3] = float("nan")       # the whole row
    x[2, 5] = float("inf")       # finite / inf = 0, inf / inf = NaN
    x[3] *= 1e-30                # squares vanish next to eps
    w = torch.ones(hidden)
    y = cb.rms_norm(x.to(DEV), w.to(DEV), eps=1e-5).cpu()
    assert torch.all(y[0] == 0) and torch.isnan(y[1]).all()
    assert torch.isnan(y[2, 5]) and torch.all(torch.cat([y[2, :5], y[2, 6:]]) == 0)
    assert torch.allclose(y[3], x[3] / 1e-5 ** 0.5, rtol=1e-5)
    q, s = cb.rms_norm(x.to(DEV), w.to(DEV), eps=1e-5, out_dtype=FP8)
    q, s = q.cpu().float(), s.cpu()
    assert torch.all(q[0] == 0) and torch.all(s[:, 0] == 2.0 ** -126)
    assert torch.isnan(q[1]).all() and torch.isnan(s[:, 1]).all()
    assert torch.isnan(s[0, 2]) and torch.isnan(q[2, :128]).all() and torch.all(q[2, 128:] == 0)
    assert torch.isfinite(q[4]).all()
    # eps 0 and a row of zeros: 0 * inf, as the formula has it
    assert torch.isnan(cb.rms_norm(x.to(DEV), w.to(DEV), eps=0.0).cpu()[0]).all()


QUANT_SHAPES = [(1, 128), (1, 1), (3, 5), (128, 128), (129, 257), (130, 264), (64, 4096), (5, 8200), (300, 72), (2, 8),
                (700, 4104), (1001, 2600)]


@pytest.mark.parametrize("rows, cols", QUANT_SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_bit_exact(rows, cols, dtype, block_rows):
    """Every step is one correctly rounded fp32 operation: equal bits."""
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    f = x.float()
    s = ref.row_scales(f) if block_rows == 1 else ref.block_scales(f)
    want = ref.to_e4m3(f, ref.spread_rows(s, cols) if block_rows == 1 else ref.spread_blocks(s, rows, cols))
    q, sd = cb.quantize_fp8(x.to(DEV), block_rows=block_rows)
    torch.cuda.synchronize()
    assert torch.equal(sd.cpu(), s)
    assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [384, 381])
def test_quantize_special_values(block_rows, cols):
    x = torch.randn(2, cols)
    x[:, :128] = 0                       # nothing but zeros (a negative one among them)
    x[0, 1] = -0.0
    x[1, 130], x[1, 131] = float("inf"), 1.0
    x[0, 300] = float("nan")
    q, s = cb.quantize_fp8(x.to(DEV), block_rows=block_rows)
    q, s = q.cpu().float(), s.cpu() if block_rows == 1 else s.cpu().t().repeat(1, 2)
    assert torch.all(s[0] == 2.0 ** -126) and torch.all(q[:, :128] == 0)
    assert torch.isinf(s[1, 1]) and torch.isnan(q[1, 130]) and q[1, 131] == 0
    assert torch.isnan(s[2, 0]) and torch.isnan(q[0, 256:]).all()
    if block_rows == 1:  # the other row's groups are their own
        assert torch.isfinite(q[0, :256]).all() and torch.isfinite(q[1, 256:]).all()
    # the smallest values: a subnormal group keeps the smallest scale
    tiny = torch.full((1, 128), 2.0 ** -140)
    q, s = cb.quantize_fp8(tiny.to(DEV))
    assert s.item() == 2.0 ** -126 and torch.all(q.cpu().float() == 0)


def test_quantize_writes_its_rows_only():
    x = torch.randn(5, 136, device=DEV)
    buf = torch.full((7 * 136,), 0x55, dtype=torch.uint8, device=DEV)
    sc = torch.full((2, 7), 3.0, device=DEV)
    out = buf[136:6 * 136].view(FP8).view(5, 136)
    cb.quantize_fp8(x, out=out, scales=sc.view(-1)[:10].view(2, 5))
    assert torch.all(buf[:136] == 0x55) and torch.all(buf[6 * 136:] == 0x55) and torch.all(sc.view(-1)[10:] == 3.0)


def test_elements_past_32_bits():
    """More than 2^31 elements: the last rows equal those of a call of their own."""
    rows, cols, last = 300000, 7200, 700
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[:1000].normal_()
    x[1000:] = x[:1000].repeat(299, 1)
    x[-last:].normal_()
    assert x.numel() > 1 << 31
    w = torch.randn(cols, device=DEV)
    assert torch.equal(cb.rms_norm(x, w)[-last:], cb.rms_norm(x[-last:], w))
    q, s = cb.rms_norm(x, w, out_dtype=FP8)
    q1, s1 = cb.rms_norm(x[-last:], w, out_dtype=FP8)
    assert torch.equal(q[-last:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[:, -last:], s1)
    q, s = cb.quantize_fp8(x)
    q1, s1 = cb.quantize_fp8(x[-last:])
    assert torch.equal(q[-last:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[:, -last:], s1)
    q, s = cb.quantize_fp8(x, block_rows=128)
    q1, s1 = cb.quantize_fp8(x[rows // 128 * 128 - 256:], block_rows=128)
    assert torch.equal(q[rows // 128 * 128 - 256:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-3:], s1)


def test_refusals():
    x, w = torch.zeros(2, 256, device=DEV), torch.ones(256, device=DEV)
    with pytest.raises(ValueError, match="contiguous"):
        cb.rms_norm(x.t().contiguous().t(), w)
    with pytest.raises(ValueError, match="CUDA"):
        cb.rms_norm(x, w.cpu())
    with pytest.raises(ValueError, match="shape"):
        cb.rms_norm(x, w[:128])
    with pytest.raises(TypeError):
        cb.rms_norm(x.double(), w)
    with pytest.raises(TypeError):
        cb.rms_norm(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        cb.rms_norm(x, w, residual_out=x)
    with pytest.raises(cb.CottusError):
        cb.rms_norm(x, w, residual=x, residual_out=x)
    with pytest.raises(ValueError, match="scales"):
        cb.rms_norm(x, w, scales=x)
    with pytest.raises(cb.CottusError):
        cb.quantize_fp8(x, block_rows=2)
    with pytest.raises(ValueError):
        cb.quantize_fp8(x[0])
    assert cb.rms_norm(x[:0], w).shape == (0, 256)
    q, s = cb.quantize_fp8(x[:0])
    assert q.shape == (0, 256) and s.shape == (2, 0)
