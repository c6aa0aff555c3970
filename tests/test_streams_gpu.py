"""Calls with a `stream` argument: their outputs come from that stream's memory
and hold, without the caller waiting for anything but that stream, what the same
call gives on the current one."""
import pytest
import torch

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"
H, HKV, D, BS, N, HIDDEN = 8, 2, 64, 16, 3, 512


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _pool_stream(t):
    """The stream whose memory holds t."""
    for seg in torch.cuda.memory_snapshot():
        if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"]:
            return seg["stream"]
    raise AssertionError("not the caching allocator's")


def _calls():
    """name -> call(stream, pool), on inputs of its own."""
    g = torch.Generator(device=DEV).manual_seed(1)

    def half(*shape):
        return torch.randn(*shape, generator=g, device=DEV).half()

    tab = cb.rope_cos_sin_table(64, D).to(DEV)
    pool = half(8 * 2 * BS * HKV * D).view(torch.int16)
    table = torch.arange(2 * N, dtype=torch.int32, device=DEV).view(N, 2)
    pos = torch.tensor([5, 17, 30], dtype=torch.int32, device=DEV)
    lens = pos + 1
    q, k, v, att = half(N, H, D), half(N, HKV, D), half(N, HKV, D), half(N, H * D)
    x, wqkv, wo = half(N, HIDDEN), half((H + 2 * HKV) * D, HIDDEN) / 16, half(HIDDEN, H * D) / 16
    res = torch.randn(N, HIDDEN, generator=g, device=DEV)
    parts, lses = torch.randn(2, N, H, D, generator=g, device=DEV), torch.randn(2, N, H, generator=g, device=DEV)
    xf = torch.randn(N, H, D, generator=g, device=DEV)
    kw = dict(num_kv_heads=HKV, head_dim=D, block_size=BS)
    return pool, {
        "paged_decode": lambda s, p: cb.paged_decode(q, p, table, lens, stream=s, **kw),
        "lse_combine": lambda s, p: cb.lse_combine(parts, lses, stream=s),
        "rope": lambda s, p: cb.rope(xf, pos, tab, stream=s),
        "rope_append_decode": lambda s, p: cb.rope_append_decode(q, k, v, pos, tab, p, table, stream=s, **kw),
        "qkv_rope_append": lambda s, p: cb.qkv_rope_append(x, wqkv, pos, tab, p, table, num_heads=H, stream=s, **kw),
        "o_proj_residual": lambda s, p: cb.o_proj_residual(att, wo, res, stream=s),
        "paged_gather": lambda s, p: cb.paged_gather(p, table, lens, max_context=32, stream=s, **kw)[0],
    }


@pytest.mark.parametrize("name", ["paged_decode", "lse_combine", "rope", "rope_append_decode", "qkv_rope_append",
                                  "o_proj_residual", "paged_gather"])
def test_outputs_belong_to_the_stream(name):
    pool, calls = _calls()
    pools = [pool.clone() for _ in range(2)]
    want = calls[name](None, pools[0])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = calls[name](side, pools[1])
    side.synchronize()
    assert _pool_stream(got) == side.cuda_stream
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)) and torch.equal(pools[0], pools[1])
