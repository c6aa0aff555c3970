"""Output types of fp8_linear and next_tokens: the one asked for, that of a given
buffer, and a refusal where the two differ."""
import pytest
import torch

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _operands():
    g = torch.Generator(device=DEV).manual_seed(2)
    return (*cb.quantize_fp8(torch.randn(5, 256, generator=g, device=DEV)),
            *cb.quantize_fp8(torch.randn(300, 256, generator=g, device=DEV) / 16, block_rows=128))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_fp8_linear_output_type(dtype):
    a = _operands()
    asked = cb.fp8_linear(*a, out_dtype=dtype)
    given = cb.fp8_linear(*a, out=torch.empty(5, 300, dtype=dtype, device=DEV))
    both = cb.fp8_linear(*a, out=torch.empty(5, 300, dtype=dtype, device=DEV), out_dtype=dtype)
    assert asked.dtype == dtype and torch.equal(asked, given) and torch.equal(asked, both)
    assert cb.fp8_linear(*a).dtype == torch.float16
    other = torch.float32 if dtype != torch.float32 else torch.float16
    buf = torch.full((5, 300), 7.0, dtype=dtype, device=DEV)
    with pytest.raises(TypeError, match="out_dtype"):
        cb.fp8_linear(*a, out=buf, out_dtype=other)
    assert torch.all(buf == 7)
    with pytest.raises(TypeError):
        cb.fp8_linear(*a, out_dtype=torch.float64)


def test_next_tokens_logits_type():
    _, _, w, ws = _operands()
    g = torch.Generator(device=DEV).manual_seed(3)
    resid, norm = torch.randn(5, 256, generator=g, device=DEV), torch.ones(256, device=DEV)
    u = torch.rand(5, generator=g, device=DEV)
    tokens, logits = cb.next_tokens(resid, norm, w, ws, u)
    assert logits.dtype == torch.float32
    buf = torch.empty(5, 300, dtype=torch.float16, device=DEV)
    half_tokens, half = cb.next_tokens(resid, norm, w, ws, u, logits=buf)
    assert half.data_ptr() == buf.data_ptr() and torch.equal(half, logits.half())
    assert torch.equal(half_tokens, cb.sample_tokens(buf, u))
