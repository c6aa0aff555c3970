"""Projections right behind the launch that writes what they read.

Kernels start before the preceding one of their stream is done and wait for it
before they read anything; a weight is no exception, since it may be what that
kernel writes (merged with an update, converted, rotated).  Each test issues a
producer and a projection on the producer's output over and over without
waiting, every time from other inputs, into the same buffers, and compares each
result, bit for bit, with that of the two calls made one at a time.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"
ROUNDS, KINDS = 60, 3


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _producers(name, rows, cols):
    """Calls that write a fp16 matrix [rows][cols] into a given buffer, one per kind of input."""
    g = _gen(17)
    out = []
    for _ in range(KINDS):
        if name == "fp8_linear":  # a weight plus a product
            x, xs = cb.quantize_fp8(_randn(g, rows, 256))
            w, ws = cb.quantize_fp8(_randn(g, cols, 256) / 16, block_rows=128)
            res = _randn(g, rows, cols)
            out.append(lambda buf, a=(x, xs, w, ws), r=res: cb.fp8_linear(*a, residual=r, out=buf))
        elif name == "rms_norm":
            x, w = _randn(g, rows, cols), 1 + 0.1 * _randn(g, cols)
            out.append(lambda buf, x=x, w=w: cb.rms_norm(x, w, out=buf))
        else:  # the projection's own fp16 output, from at most 64 rows
            x, w, res = _randn(g, rows, 256).half(), (_randn(g, cols, 256) / 16).half(), _randn(g, rows, cols)
            out.append(lambda buf, a=(x, w, res): cb.o_proj_residual(*a, out=buf))
    return out


@pytest.mark.parametrize("producer", ["fp8_linear", "rms_norm", "o_proj_residual"])
@pytest.mark.parametrize("tokens", [1, 20, 64])
def test_o_proj_weight_written_just_before(producer, tokens):
    rows, cols = 1024, 2048
    make = _producers(producer, rows, cols)
    g = _gen(3)
    x, res = _randn(g, tokens, cols).half(), _randn(g, tokens, rows)
    weight = torch.zeros(rows, cols, dtype=torch.float16, device=DEV)
    want = []
    for f in make:
        f(weight)
        torch.cuda.synchronize()
        want.append(cb.o_proj_residual(x, weight, res))
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    outs = []
    for i in range(ROUNDS):
        make[i % KINDS](weight)
        outs.append(cb.o_proj_residual(x, weight, res))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % KINDS]), i


@pytest.mark.parametrize("producer", ["fp8_linear", "rms_norm"])
def test_qkv_weight_written_just_before(producer):
    H, HKV, D, BS, n, hidden = 8, 2, 64, 16, 5, 1024
    make = _producers(producer, (H + 2 * HKV) * D, hidden)
    g = _gen(4)
    x = _randn(g, n, hidden).half()
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    tab = cb.rope_cos_sin_table(BS, D).to(DEV)
    table = torch.arange(n, dtype=torch.int32, device=DEV).view(n, 1)
    pool = torch.zeros(n * 2 * BS * HKV * D, dtype=torch.int16, device=DEV)
    weight = torch.zeros((H + 2 * HKV) * D, hidden, dtype=torch.float16, device=DEV)

    def project():
        return cb.qkv_rope_append(x, weight, pos, tab, pool, table, num_heads=H, num_kv_heads=HKV, head_dim=D,
                                  block_size=BS)

    want = []
    for f in make:
        f(weight)
        torch.cuda.synchronize()
        want.append((project(), pool.clone()))
        torch.cuda.synchronize()
    outs = []
    for i in range(ROUNDS):
        make[i % KINDS](weight)
        outs.append((project(), pool.clone()))
    torch.cuda.synchronize()
    for i, (q, p) in enumerate(outs):
        assert torch.equal(q, want[i % KINDS][0]) and torch.equal(p, want[i % KINDS][1]), i
