"""The scale ring of the block-scaled product over many passes.

Scales go to a ring in shared memory, a few groups at once, and its slots are
given back by the warps that have read them.  A slot that is written again too
early, or read too late, shows as another group's scale: here each group's and
each row's scales are drawn apart, and there are many more groups, and tiles per
CTA, than the ring has slots.

Values up to 4, scales 1 or 2: a sum of k products is at most 64 k < 2^24 and a
whole number, so every order of additions in fp32 gives it exactly.
"""
import pytest
import torch

import lowp_ref as ref

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _case(m, n, k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEV).float()

    x, w = ints(-4, 5, m, k), ints(-4, 5, n, k)
    xs, ws = 2 ** ints(0, 2, ref.groups(k), m), 2 ** ints(0, 2, ref.groups(n), ref.groups(k))
    want = torch.zeros(m, n, dtype=torch.float64, device=DEV)
    for b in range(ref.groups(k)):
        c = slice(b * 128, (b + 1) * 128)
        rows = ws[:, b].double().repeat_interleave(128)[:n]
        want.addmm_(x[:, c].double() * xs[b].double()[:, None], (w[:, c].double() * rows[:, None]).t())
    return x.to(FP8), xs, w.to(FP8), ws, want.float()


# each number of rows per CTA with several tiles per CTA, with splits, and the
# pairs; groups that are no multiple of what the ring takes at once
@pytest.mark.parametrize("m, n, k", [(13, 40000, 8336), (29, 40000, 8336), (60, 40000, 8336), (128, 40000, 8336),
                                     (30, 640, 60000), (120, 384, 60000), (1500, 8200, 8336), (300, 20000, 30000)])
def test_many_passes_of_the_scale_ring(m, n, k):
    x, xs, w, ws, want = _case(m, n, k, m + n)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    outs = [cb.fp8_linear(x, xs, w, ws, out_dtype=torch.float32, status=st) for _ in range(10)]
    torch.cuda.synchronize()
    assert int(st.item()) == 0
    for o in outs:
        assert torch.equal(o, want)
