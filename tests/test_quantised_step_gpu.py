"""The norm, 8-bit and sampling operators as a decode step uses them together:
an 8-bit attention block and the way from the residual stream to the next token
over a running DecodeBatch, in CUDA graphs, on several streams and after one
another without waiting.

The blocks are compositions: their results equal, bit for bit, those of the
operators called one by one (each is held to its definition elsewhere), and
their attention is held to the oracle from the projections on.
"""
import os
import pathlib
import subprocess
import sys

import numpy as np
import pytest
import torch

import lowp_ref as ref
from helpers import TOL_F16

pytestmark = pytest.mark.gpu

cb = pytest.importorskip("cottus_b200")

DEV = "cuda"
FP8 = torch.float8_e4m3fn
H, HKV, D, BS, LAYERS, HIDDEN, VOCAB = 8, 2, 64, 16, 2, 512, 1000


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _weights(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def q(rows, cols):
        return cb.quantize_fp8(torch.randn(rows, cols, generator=g, device=DEV) / cols ** 0.5, block_rows=128)

    layers = [dict(norm=1 + 0.1 * torch.randn(HIDDEN, generator=g, device=DEV), qkv=q((H + 2 * HKV) * D, HIDDEN),
                   o=q(HIDDEN, H * D)) for _ in range(LAYERS)]
    return layers, 1 + 0.1 * torch.randn(HIDDEN, generator=g, device=DEV), q(VOCAB, HIDDEN)


def _block(batch, resid, w, pool, tab, layer):
    return cb.attention_block_fp8(batch, resid, w["norm"], *w["qkv"], *w["o"], pool, tab, num_heads=H, num_kv_heads=HKV,
                                  head_dim=D, num_layers=LAYERS, layer=layer)


def test_decode_loop_with_joins(oracle):
    """Twelve steps of two layers over a batch that grows: residual stream, pool and tokens against the operators called
    one by one; attention against the oracle."""
    layers, norm, head = _weights(1)
    emb = torch.randn(VOCAB, HIDDEN, device=DEV)
    tab = cb.rope_cos_sin_table(64, D).to(DEV)
    blocks = 24
    pool = torch.zeros(blocks * 2 * LAYERS * BS * HKV * D, dtype=torch.int16, device=DEV)
    pool2 = pool.clone()
    hpool = np.zeros(pool.numel(), np.uint16)
    batch = cb.DecodeBatch(blocks, BS, 6, 4, device=DEV)
    last = {}
    rng = np.random.default_rng(3)
    for step in range(12):
        if step % 3 == 0:
            batch.add(step)
            last[step] = int(rng.integers(VOCAB))
        batch.begin_step()
        rows = batch.rows()
        n = len(rows)
        resid = emb[[last[r] for r in rows]].contiguous()
        one = resid.clone()
        u = torch.rand(n, device=DEV)
        for layer, w in enumerate(layers):
            att = _block(batch, resid, w, pool, tab, layer)
            # the same, one operator after the other
            h, hs = cb.rms_norm(one, w["norm"], out_dtype=FP8)
            wq, ws = w["qkv"]
            q, k, v = (cb.fp8_linear(h, hs, wq[a:b], ws[a // 128:b // 128]) for a, b in
                       ((0, H * D), (H * D, (H + HKV) * D), ((H + HKV) * D, (H + 2 * HKV) * D)))
            att2 = cb.rope_append_decode(q.view(n, H, D), k.view(n, HKV, D), v.view(n, HKV, D), batch.positions[:n], tab,
                                         pool2, batch.block_table[:n], num_kv_heads=HKV, head_dim=D, block_size=BS,
                                         num_layers=LAYERS, layer=layer)
            a8, a8s = cb.quantize_fp8(att2.view(n, H * D))
            one = cb.fp8_linear(a8, a8s, *w["o"], residual=one, out_dtype=torch.float32)
            assert torch.equal(att, att2.view(n, H * D)) and torch.equal(resid, one)
            qh, kh, vh = (t.float().cpu().numpy() for t in (q, k, v))
            for r, sid in enumerate(rows):
                _, pos, blk = batch.sequence(sid)
                oracle.kv_append(hpool, oracle.rope(kh[r].reshape(HKV, D), pos, HKV, D), vh[r].reshape(HKV, D), blk, pos, layer,
                                 HKV, D, BS, LAYERS)
                want = oracle.paged_attention(oracle.rope(qh[r].reshape(H, D), pos, H, D), hpool, blk, pos + 1, layer, H, HKV,
                                              D, BS, LAYERS)
                assert np.max(np.abs(att[r].float().cpu().numpy() - np.asarray(want).reshape(-1))) <= TOL_F16
        tokens, logits = cb.next_tokens(resid, norm, *head, u, temperature=torch.full((n,), 0.8, device=DEV),
                                        top_k=torch.full((n,), 40, dtype=torch.int32, device=DEV),
                                        top_p=torch.full((n,), 0.95, device=DEV))
        for r, sid in enumerate(rows):
            want, _, _ = ref.sample(logits[r].cpu().numpy(), float(u[r]), float(np.float32(0.8)), 40, float(np.float32(0.95)))
            assert want is None or int(tokens[r]) == want
            last[sid] = int(tokens[r])
        batch.end_step()
    assert torch.equal(pool, pool2)
    assert np.array_equal(pool.cpu().numpy().view(np.uint16), hpool)


def test_blocks_refuse_wrong_shapes():
    layers, _, _ = _weights(2)
    batch = cb.DecodeBatch(4, BS, 2, 2, device=DEV)
    batch.add(0)
    tab = cb.rope_cos_sin_table(32, D).to(DEV)
    pool = torch.zeros(4 * 2 * LAYERS * BS * HKV * D, dtype=torch.int16, device=DEV)
    w = layers[0]
    with pytest.raises(ValueError, match="one row per"):
        _block(batch, torch.zeros(2, HIDDEN, device=DEV), w, pool, tab, 0)
    with pytest.raises(ValueError, match="multiples of 128"):
        cb.attention_block_fp8(batch, torch.zeros(1, HIDDEN, device=DEV), w["norm"], *w["qkv"], *w["o"], pool, tab,
                               num_heads=H, num_kv_heads=1, head_dim=D)
    with pytest.raises(ValueError, match="rows"):
        cb.attention_block_fp8(batch, torch.zeros(1, HIDDEN, device=DEV), w["norm"], *w["o"], *w["o"], pool, tab,
                               num_heads=H, num_kv_heads=HKV, head_dim=D)


@pytest.mark.parametrize("rows", [1, 5, 40, 150])
def test_graph_replay(rows):
    """norm -> projection -> sampling captured once and replayed on new inputs: the results of eager calls."""
    _, norm, head = _weights(4)
    resid, u = torch.randn(rows, HIDDEN, device=DEV), torch.rand(rows, device=DEV)
    top_p, k = torch.full((rows,), 0.9, device=DEV), torch.full((rows,), 50, dtype=torch.int32, device=DEV)
    kinds = (dict(), dict(top_k=k), dict(top_p=top_p), dict(top_k=k, top_p=top_p))
    for kw in kinds:
        cb.next_tokens(resid, norm, *head, u, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [cb.next_tokens(resid, norm, *head, u, **kw) for kw in kinds]
    for seed in range(3):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        resid.copy_(torch.randn(rows, HIDDEN, generator=gen, device=DEV))
        u.copy_(torch.rand(rows, generator=gen, device=DEV))
        g.replay()
        g.replay()  # twice in a row: no state is left behind
        torch.cuda.synchronize()
        for (tok, logits), kw in zip(outs, kinds):
            want, want_logits = cb.next_tokens(resid, norm, *head, u, **kw)
            assert torch.equal(tok, want) and torch.equal(logits, want_logits)


def test_two_streams_at_once():
    """Calls on two streams that overlap, on a stream handed over, and two graphs replayed side by side."""
    _, norm, head = _weights(5)
    data = [(torch.randn(24, HIDDEN, device=DEV), torch.rand(24, device=DEV)) for _ in range(2)]
    want = [cb.next_tokens(r, norm, *head, u, top_p=torch.full((24,), 0.8, device=DEV)) for r, u in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    p = torch.full((24,), 0.8, device=DEV)
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cb.next_tokens(*(data[i][0], norm), *head, data[i][1], top_p=p))
    torch.cuda.synchronize()
    for i in range(2):
        for tok, logits in got[i]:
            assert torch.equal(tok, want[i][0]) and torch.equal(logits, want[i][1])
    logits = torch.empty(24, VOCAB, device=DEV)
    tok, _ = cb.next_tokens(data[0][0], norm, *head, data[0][1], top_p=p, logits=logits, stream=streams[1])
    streams[1].synchronize()
    assert torch.equal(tok, want[0][0]) and torch.equal(logits, want[0][1])
    graphs = []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = cb.next_tokens(data[i][0], norm, *head, data[i][1], top_p=p)
        graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i, (_, (tok, logits)) in enumerate(graphs):
        assert torch.equal(tok, want[i][0]) and torch.equal(logits, want[i][1])


@pytest.mark.parametrize("rows", [1, 5, 16, 70])
def test_weights_written_just_before(rows):
    """A projection right behind the kernel that writes its weight, and behind the one that writes its input, over and
    over without waiting: it may prefetch, but not read, before they are done."""
    g = torch.Generator(device=DEV).manual_seed(6)
    ws = [torch.randn(1024, HIDDEN, generator=g, device=DEV) for _ in range(3)]
    xs = [torch.randn(rows, HIDDEN, generator=g, device=DEV) for _ in range(3)]
    want = []
    for w, x in zip(ws, xs):
        want.append(cb.fp8_linear(*cb.quantize_fp8(x), *cb.quantize_fp8(w, block_rows=128), out_dtype=torch.float32))
        torch.cuda.synchronize()
    wq, wsc = torch.empty(1024, HIDDEN, dtype=FP8, device=DEV), torch.empty(8, HIDDEN // 128, device=DEV)
    xq, xsc = torch.empty(rows, HIDDEN, dtype=FP8, device=DEV), torch.empty(HIDDEN // 128, rows, device=DEV)
    outs = []
    for i in range(60):
        cb.quantize_fp8(xs[i % 3], out=xq, scales=xsc)
        cb.quantize_fp8(ws[i % 3], block_rows=128, out=wq, scales=wsc)
        outs.append(cb.fp8_linear(xq, xsc, wq, wsc, out_dtype=torch.float32))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 3]), i


def _long_batches(n, tokens):
    """Batches of one long sequence each, with room for what their split decode needs."""
    out = []
    for i in range(n):
        b = cb.DecodeBatch(tokens // BS + 2, BS, 1, tokens // BS + 2, device=DEV)
        b.add(i)
        for _ in range(tokens):
            b.begin_step()
            b.end_step()
        b.begin_step()
        out.append(b)
    torch.cuda.synchronize()
    return out


def test_blocks_of_two_batches_at_once():
    """Two batches with a long context each, on two streams, by the stream argument, and captured as the first call of
    their batch: each has its own workspace and its temporaries from its own stream's pool."""
    tokens = 1500
    layers, _, _ = _weights(7)
    tab = cb.rope_cos_sin_table(tokens + BS, D).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(8)
    pools, want, start = [], [], []
    batches = _long_batches(2, tokens)
    for b in batches:
        pools.append(torch.randn(b.num_blocks * 2 * LAYERS * BS * HKV * D, generator=g, device=DEV).half().view(torch.int16))
        start.append(torch.randn(1, HIDDEN, generator=g, device=DEV))
        r = start[-1].clone()
        att = [_block(b, r, w, pools[-1], tab, i) for i, w in enumerate(layers)]
        want.append((att, r))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    rows = [[s.clone() for _ in range(20)] for s in start]
    got = [[], []]
    torch.cuda.synchronize()
    for j in range(20):
        for i, s in enumerate(streams):
            for layer, w in enumerate(layers):
                got[i].append(cb.attention_block_fp8(batches[i], rows[i][j], w["norm"], *w["qkv"], *w["o"], pools[i], tab,
                                                     num_heads=H, num_kv_heads=HKV, head_dim=D, num_layers=LAYERS, layer=layer,
                                                     stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        for j in range(20):
            assert torch.equal(rows[i][j], want[i][1])
            for layer in range(LAYERS):
                assert torch.equal(got[i][j * LAYERS + layer], want[i][0][layer])
    # captured before their batch ever ran eagerly
    graphs = []
    for i, b in enumerate(_long_batches(2, tokens)):
        r = start[i].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for layer, w in enumerate(layers):
                _block(b, r, w, pools[i], tab, layer)
        graphs.append((graph, r, b))
    torch.cuda.synchronize()
    for _ in range(10):
        for i, (graph, r, _) in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                r.copy_(start[i])
                graph.replay()
    torch.cuda.synchronize()
    for i, (_, r, _) in enumerate(graphs):
        assert torch.equal(r, want[i][1])


def test_first_call_inside_a_capture():
    """A process whose first call of each operator is captured: what a call sets up once is no stream work."""
    script = """
import torch, cottus_b200 as cb
dev = "cuda"
r, u = torch.randn(3, 256, device=dev), torch.rand(3, device=dev)
n = torch.ones(256, device=dev)
wide = torch.randn(300, 256, device=dev)
p = torch.full((3,), 0.9, device=dev)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    w, ws = cb.quantize_fp8(torch.ones(5000, 256, device=dev) * u[0] + n, block_rows=128)
    x, xs = cb.quantize_fp8(wide)
    y = cb.fp8_linear(x, xs, w, ws)
    t, logits = cb.next_tokens(r, n, w, ws, u, top_p=p)
g.replay()
torch.cuda.synchronize()
t2, l2 = cb.next_tokens(r, n, w, ws, u, top_p=p)
assert torch.equal(t, t2) and torch.equal(logits, l2) and torch.equal(y, cb.fp8_linear(x, xs, w, ws))
print("same")
"""
    root = pathlib.Path(cb.__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": str(root)})
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


def test_empty_batch():
    """A step in which no sequence is active."""
    layers, norm, head = _weights(9)
    batch = cb.DecodeBatch(4, BS, 2, 2, device=DEV)
    batch.begin_step()
    tab = cb.rope_cos_sin_table(32, D).to(DEV)
    pool = torch.zeros(4 * 2 * LAYERS * BS * HKV * D, dtype=torch.int16, device=DEV)
    resid = torch.zeros(0, HIDDEN, device=DEV)
    assert _block(batch, resid, layers[0], pool, tab, 0).shape == (0, H * D)
    tokens, logits = cb.next_tokens(resid, norm, *head, torch.zeros(0, device=DEV))
    assert tokens.shape == (0,) and logits.shape == (0, VOCAB)
    torch.cuda.synchronize()
