"""The norm, 8-bit and sampling entry points without a GPU: every refusal
happens before CUDA is touched, and an empty call is a successful no-op."""
import ctypes as C

import pytest
import torch

cb = pytest.importorskip("cottus_b200")
from cottus_b200 import _lib  # noqa: E402

BAD, UNSUP, OK = _lib.COTTUS_ERR_INVALID_ARGUMENT, _lib.COTTUS_ERR_UNSUPPORTED, _lib.COTTUS_OK
MB = 1 << 20


def _norm(**kw):
    p = _lib.RmsNormParams()
    p.x, p.weight, p.out = 1 * MB, 2 * MB, 3 * MB
    p.rows, p.hidden, p.x_dtype, p.out_dtype, p.eps = 4, 256, _lib.F16, _lib.F16, 1e-5
    for k, v in kw.items():
        setattr(p, k, v)
    return _lib.lib().cottus_rms_norm(C.byref(p), None)


def _quant(**kw):
    p = _lib.QuantizeParams()
    p.x, p.out, p.scales = 1 * MB, 2 * MB, 3 * MB
    p.rows, p.cols, p.x_dtype, p.block_rows = 4, 256, _lib.F32, 1
    for k, v in kw.items():
        setattr(p, k, v)
    return _lib.lib().cottus_quantize_fp8(C.byref(p), None)


def _linear(**kw):
    p = _lib.Fp8LinearParams()
    p.x, p.x_scales, p.weight, p.w_scales, p.out = 1 * MB, 2 * MB, 3 * MB, 4 * MB, 5 * MB
    p.rows, p.out_features, p.in_features, p.out_dtype = 4, 256, 512, _lib.F32
    for k, v in kw.items():
        setattr(p, k, v)
    return _lib.lib().cottus_fp8_linear(C.byref(p), None)


def _sample(**kw):
    p = _lib.SampleParams()
    p.logits, p.uniforms, p.tokens = 1 * MB, 2 * MB, 3 * MB
    p.batch, p.vocab, p.dtype = 4, 1000, _lib.F32
    for k, v in kw.items():
        setattr(p, k, v)
    return _lib.lib().cottus_sample_tokens(C.byref(p), None)


def _message():
    return _lib.lib().cottus_last_error().decode()


@pytest.mark.parametrize("kw, code, text", [
    (dict(rows=-1), BAD, "rows"), (dict(hidden=0), BAD, "hidden"), (dict(x_dtype=_lib.E4M3), BAD, "x dtype"),
    (dict(out_dtype=9), BAD, "out dtype"), (dict(eps=-1.0), BAD, "eps"), (dict(eps=float("nan")), BAD, "eps"),
    (dict(eps=float("inf")), BAD, "eps"), (dict(x=None), BAD, "NULL"), (dict(weight=None), BAD, "NULL"),
    (dict(out=None), BAD, "NULL"), (dict(residual=4 * MB), BAD, "residual_out"),
    (dict(residual_out=4 * MB), BAD, "residual_out"), (dict(scales=4 * MB), BAD, "scales"),
    (dict(out_dtype=_lib.E4M3), BAD, "scales"), (dict(rows=1 << 31), UNSUP, "rows"),
    (dict(out=1 * MB + 512), BAD, "overlaps"), (dict(out=1 * MB, out_dtype=_lib.F32), BAD, "overlaps"),
    (dict(out=2 * MB), BAD, "overlaps"), (dict(residual=4 * MB, residual_out=4 * MB + 1024), BAD, "overlaps"),
    (dict(residual=3 * MB, residual_out=5 * MB), BAD, "overlaps"),
    (dict(residual=4 * MB, residual_out=3 * MB), BAD, "overlaps"),
    (dict(residual=4 * MB, residual_out=1 * MB), BAD, "overlaps"),
    (dict(out_dtype=_lib.E4M3, scales=3 * MB + 256), BAD, "overlaps"), (dict(x=1 * MB + 1), BAD, "aligned"),
    (dict(weight=2 * MB + 2), BAD, "aligned"),
])
def test_rms_norm_refusals(kw, code, text):
    assert _norm(**kw) == code
    assert text in _message()


@pytest.mark.parametrize("kw, code, text", [
    (dict(rows=-1), BAD, "rows"), (dict(cols=0), BAD, "cols"), (dict(x_dtype=_lib.E4M3), BAD, "dtype"),
    (dict(block_rows=64), BAD, "block_rows"), (dict(x=None), BAD, "NULL"), (dict(out=None), BAD, "NULL"),
    (dict(scales=None), BAD, "NULL"), (dict(out=1 * MB), BAD, "overlaps"), (dict(scales=2 * MB + 4), BAD, "overlaps"),
    (dict(scales=1 * MB + 4), BAD, "overlaps"), (dict(x=1 * MB + 2), BAD, "aligned"),
    (dict(scales=3 * MB + 2), BAD, "aligned"), (dict(rows=1 << 40, x=1 << 60), UNSUP, "rows"),
    (dict(rows=65536 * 128, block_rows=128), UNSUP, "rows"),
])
def test_quantize_refusals(kw, code, text):
    assert _quant(**kw) == code
    assert text in _message()


@pytest.mark.parametrize("kw, code, text", [
    (dict(rows=-1), BAD, "rows"), (dict(out_features=0), BAD, "out_features"), (dict(in_features=0), BAD, "in_features"),
    (dict(out_dtype=_lib.E4M3), BAD, "dtype"), (dict(in_features=520), UNSUP, "16"), (dict(x=None), BAD, "NULL"),
    (dict(x_scales=None), BAD, "NULL"), (dict(weight=None), BAD, "NULL"), (dict(w_scales=None), BAD, "NULL"),
    (dict(out=None), BAD, "NULL"), (dict(x=1 * MB + 8), BAD, "16-byte"), (dict(weight=3 * MB + 8), BAD, "16-byte"),
    (dict(out=5 * MB + 2), BAD, "aligned"), (dict(residual=6 * MB + 2), BAD, "aligned"), (dict(out=1 * MB), BAD, "overlaps"),
    (dict(out=3 * MB + 64), BAD, "overlaps"), (dict(out=2 * MB), BAD, "overlaps"), (dict(out=4 * MB), BAD, "overlaps"),
    (dict(residual=5 * MB, out_dtype=_lib.F16), BAD, "overlaps"), (dict(residual=5 * MB + 16), BAD, "overlaps"),
])
def test_fp8_linear_refusals(kw, code, text):
    assert _linear(**kw) == code
    assert text in _message()


@pytest.mark.parametrize("kw, code, text", [
    (dict(batch=-1), BAD, "batch"), (dict(vocab=0), BAD, "vocab"), (dict(dtype=_lib.E4M3), BAD, "dtype"),
    (dict(vocab=327681), UNSUP, "vocab"), (dict(logits=None), BAD, "NULL"), (dict(uniforms=None), BAD, "NULL"),
    (dict(tokens=None), BAD, "NULL"), (dict(logits=1 * MB + 2), BAD, "aligned"), (dict(top_k=4 * MB + 1), BAD, "aligned"),
    (dict(tokens=1 * MB), BAD, "overlaps"), (dict(tokens=2 * MB + 4), BAD, "overlaps"),
    (dict(logprobs=3 * MB + 4), BAD, "overlaps"), (dict(temperature=4 * MB, logprobs=4 * MB), BAD, "overlaps"),
])
def test_sample_refusals(kw, code, text):
    assert _sample(**kw) == code
    assert text in _message()


def test_null_params_and_empty_calls():
    L = _lib.lib()
    for fn in (L.cottus_rms_norm, L.cottus_quantize_fp8, L.cottus_fp8_linear, L.cottus_sample_tokens):
        assert fn(None, None) == BAD
    assert _norm(rows=0, x=None, out=None) == OK
    assert _quant(rows=0, x=None) == OK
    assert _linear(rows=0, x=None) == OK
    assert _sample(batch=0, logits=None) == OK
    # a shape that no non-empty call could have is refused even when the call is empty
    assert _linear(rows=0, in_features=24) == UNSUP


def test_the_attention_calls_do_not_take_the_new_types():
    p = _lib.PagedDecodeParams()
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim, p.block_size, p.num_layers = 1, 4, 2, 64, 16, 1
    for t in (_lib.BF16, _lib.E4M3):
        p.q_dtype, p.out_dtype = t, _lib.F16
        assert _lib.lib().cottus_paged_decode(C.byref(p), None) == BAD
        assert "dtype" in _message()


def test_host_tensors_are_refused():
    if not torch.cuda.is_available():
        pytest.skip("the current device is asked for first")
    x = torch.zeros(2, 128)
    with pytest.raises(ValueError):
        cb.rms_norm(x, torch.ones(128))


WIDE = (1 << 30) + 16


@pytest.mark.parametrize("call", [lambda: _norm(rows=1, hidden=WIDE), lambda: _norm(rows=1, hidden=(1 << 31) - 8),
                                  lambda: _quant(rows=1, cols=WIDE), lambda: _quant(rows=1, cols=(1 << 31) - 1, block_rows=128),
                                  lambda: _quant(rows=(1 << 63) - 1, cols=1, block_rows=128, x=1 << 60),
                                  lambda: _linear(rows=WIDE, in_features=16), lambda: _linear(rows=1, out_features=(1 << 31) - 1),
                                  lambda: _linear(rows=1, in_features=WIDE)])
def test_sizes_that_32_bit_columns_cannot_round_up(call):
    assert call() == UNSUP
    assert "too" in _message()


def test_sizes_past_32_bits_are_not_cut():
    """ctypes keeps the lower 32 bits of a larger size; the wrappers refuse it."""
    from cottus_b200 import ops
    assert ops._i32((1 << 31) - 1, "rows") == (1 << 31) - 1
    for n in (1 << 31, (1 << 32) + 5, -1):
        with pytest.raises(ValueError, match="rows"):
            ops._i32(n, "rows")
