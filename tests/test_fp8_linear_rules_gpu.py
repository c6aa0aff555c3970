"""fp8_linear at the borders between its kernels for few rows: all CTAs of the
thin kernel resident at once or in two waves, one to five groups per warp, the
second of two nearly full or not, and the narrow tile on the other sides.

The bound is that of test_fp8_linear_gpu: 128 products and the groups' sums, each
addition off by a step of fp32 at most, and the output's rounding.
"""
import pytest
import torch

from test_fp8_linear_gpu import _check, _quantised

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("m", [1, 8, 9])
@pytest.mark.parametrize("n, k", [(4736, 8192), (4736, 8208), (4737, 2048), (4737, 2064), (5120, 2560), (4752, 3456),
                                  (4752, 3472), (4752, 4096), (4752, 4112), (5120, 5120), (9472, 4096), (9473, 1024)])
def test_borders_of_the_thin_kernel(m, n, k):
    x, xs, w, ws = _quantised(m, n, k, m + n + k)
    res = torch.randn(m, n, generator=torch.Generator().manual_seed(k))
    got = cb.fp8_linear(*(t.to(DEV) for t in (x, xs, w, ws)), residual=res.to(DEV), out_dtype=torch.float32)
    _check(got, x, xs, w, ws, res)
