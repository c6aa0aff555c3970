"""Torch-facing wrappers over the C ABI.

torch is used only for device memory and the current CUDA stream; all
arithmetic runs in libcottus_b200.so.  Tensors must be contiguous CUDA
tensors on the current device (the block pool helpers are host-only).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools

import torch

from . import _lib
from ._lib import (BF16, E4M3, F16, F32, CottusError, DecodeBatchDesc, DecodeStepParams, Fp8LinearParams,
                   LseCombineParams, PagedDecodeParams, OProjParams, QkvParams, QuantizeParams, RmsNormParams,
                   SampleParams, check, lib)

_DT = {torch.float32: F32, torch.float16: F16}
_FP8 = torch.float8_e4m3fn
_DT_WIDE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}  # norm, 8-bit and sampling operators


def _dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; use float32 or float16") from None


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream(stream):
    if stream is None:
        stream = torch.cuda.current_stream()
    return C.c_void_p(stream.cuda_stream)


def _require(t: torch.Tensor, name: str, dtype=None):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _on(stream):
    """The context in which the caching allocator serves `stream` (None: the current one)."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _streamed(call):
    """A call with a `stream` argument makes everything on that stream: what it allocates comes from that stream's memory
    (of another's it might hold what that one still reads), and what it clears is cleared before it is written."""

    @functools.wraps(call)
    def on_its_stream(*args, stream=None, **kw):
        if stream is None:
            return call(*args, **kw)
        if stream.device_index != torch.cuda.current_device():
            raise ValueError(f"the stream is on cuda:{stream.device_index}, the current device is "
                             f"cuda:{torch.cuda.current_device()}")
        with _on(stream):
            return call(*args, stream=stream, **kw)

    return on_its_stream


def _capturing(device: torch.device) -> bool:
    """Whether what the current stream does goes into a graph."""
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class _Scratch:
    """Scratch memory that grows with what calls need.  Every buffer stays: a captured graph, or a kernel still running on
    another stream, may hold an earlier, smaller one (each is at least twice the one before, so that they add up to
    little).  A buffer made while a graph is captured is that graph's own, and with `cleared` cleared at each replay: until
    the first replay nothing has written it, so no other call may have it."""

    def __init__(self, device: torch.device, cleared: bool):
        self.device, self.make, self.buffers = device, torch.zeros if cleared else torch.empty, []

    def get(self, nbytes: int, stream=None) -> torch.Tensor:
        """At least nbytes, allocated (and cleared) on the stream that uses them."""
        last = self.buffers[-1].numel() if self.buffers else 1 << 19
        if self.buffers and last >= nbytes:
            return self.buffers[-1]
        with _on(stream):
            capturing = _capturing(self.device)
            buf = self.make(max(nbytes, 0 if capturing else 2 * last), dtype=torch.uint8, device=self.device)
        if not capturing:
            self.buffers.append(buf)
        return buf


_WS: dict = {}


def workspace(nbytes: int, device: torch.device, kind: str = "decode", stream=None) -> torch.Tensor:
    """Cached scratch buffer (a convenience of this Python layer; the C ABI
    itself only takes caller-provided workspace).  One buffer per kind: the
    decode kernels keep the counter words at the start of theirs at zero
    between calls, while the projections ("proj") overwrite all of theirs
    with split partials, so the two never share one."""
    key = (device.type, device.index, kind)
    if key not in _WS:
        _WS[key] = _Scratch(device, cleared=kind == "decode")
    return _WS[key].get(nbytes, stream)


def make_decode_params(out, query, kv_pool, block_table, context_lens, *, num_kv_heads, head_dim, block_size,
                       num_layers=1, layer=0, num_physical_blocks=None, scale=0.0, lse_out=None, status=None,
                       ws=None) -> PagedDecodeParams:
    B, H = query.shape[0], query.shape[1]
    if num_physical_blocks is None:
        per_block = 2 * num_layers * block_size * num_kv_heads * head_dim
        num_physical_blocks = kv_pool.numel() // per_block if per_block > 0 else 0
    p = PagedDecodeParams()
    p.out, p.query, p.kv_pool = out.data_ptr(), query.data_ptr(), kv_pool.data_ptr()
    p.block_table, p.context_lens = block_table.data_ptr(), context_lens.data_ptr()
    p.num_physical_blocks = int(num_physical_blocks)
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim = B, H, num_kv_heads, head_dim
    p.block_size, p.num_layers, p.layer = block_size, num_layers, layer
    p.max_blocks_per_seq = block_table.shape[1] if block_table.dim() == 2 else 0
    p.q_dtype, p.out_dtype = _dtype_code(query), _dtype_code(out)
    p.scale = float(scale)
    p.lse_out = lse_out.data_ptr() if lse_out is not None else None
    p.status = status.data_ptr() if status is not None else None
    if ws is not None:
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
    return p


@_streamed
def paged_decode(query: torch.Tensor, kv_pool: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
                 *, num_kv_heads: int, head_dim: int, block_size: int, num_layers: int = 1, layer: int = 0,
                 out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, scale: float = 0.0,
                 lse_out: torch.Tensor | None = None, status: torch.Tensor | None = None,
                 num_physical_blocks: int | None = None, stream=None) -> torch.Tensor:
    """Batched paged decode attention (cottus_paged_decode)."""
    _require(query, "query")
    _require(kv_pool, "kv_pool")
    _require(block_table, "block_table", torch.int32)
    _require(context_lens, "context_lens", torch.int32)
    if out is None:
        out = torch.empty(query.shape, dtype=out_dtype or query.dtype, device=query.device)
    p = make_decode_params(out, query, kv_pool, block_table, context_lens, num_kv_heads=num_kv_heads,
                           head_dim=head_dim, block_size=block_size, num_layers=num_layers, layer=layer,
                           num_physical_blocks=num_physical_blocks, scale=scale, lse_out=lse_out, status=status)
    need = lib().cottus_paged_decode_workspace_size(C.byref(p))
    if need:
        ws = workspace(need, query.device, stream=stream)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().cottus_paged_decode(C.byref(p), _stream(stream)))
    return out


def decode_workspace_size(p: PagedDecodeParams) -> int:
    return int(lib().cottus_paged_decode_workspace_size(C.byref(p)))


@_streamed
def lse_combine(partial_out: torch.Tensor, partial_lse: torch.Tensor, *, out: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.float32, lse_out: torch.Tensor | None = None, stream=None):
    """Merge [P][B][H][D] normalised partials with their [P][B][H] LSEs."""
    _require(partial_out, "partial_out", torch.float32)
    _require(partial_lse, "partial_lse", torch.float32)
    P, B, H, D = partial_out.shape
    if out is None:
        out = torch.empty((B, H, D), dtype=out_dtype, device=partial_out.device)
    p = LseCombineParams()
    p.out, p.partial_out, p.partial_lse = out.data_ptr(), partial_out.data_ptr(), partial_lse.data_ptr()
    p.lse_out = lse_out.data_ptr() if lse_out is not None else None
    p.num_parts, p.batch, p.num_heads, p.head_dim, p.out_dtype = P, B, H, D, _dtype_code(out)
    check(lib().cottus_lse_combine(C.byref(p), _stream(stream)))
    return out


def rope_cos_sin_table(max_position: int, head_dim: int, theta: float = 10000.0) -> torch.Tensor:
    """Host (cos, sin) table [max_position][head_dim/2][2] from the reference formula."""
    t = torch.empty((max_position, head_dim // 2, 2), dtype=torch.float32)
    check(lib().cottus_rope_cos_sin_fill(C.c_void_p(t.data_ptr()), max_position, head_dim, float(theta)))
    return t


@_streamed
def rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, *, out: torch.Tensor | None = None,
         stream=None) -> torch.Tensor:
    """RoPE of fp32 x[num_tokens][num_heads][head_dim] (in place when out is x)."""
    _require(x, "x", torch.float32)
    _require(positions, "positions", torch.int32)
    _require(cos_sin, "cos_sin", torch.float32)
    T, H, D = x.shape
    if out is None:
        out = torch.empty_like(x)
    check(lib().cottus_rope(_ptr(out), _ptr(x), _ptr(positions), T, H, D, _ptr(cos_sin), cos_sin.shape[0],
                            _stream(stream)))
    return out


def make_step_params(query, key, value, positions, cos_sin, kv_pool, block_table, *, num_kv_heads, head_dim,
                     block_size, num_layers=1, layer=0, num_physical_blocks=None, query_out=None, out=None,
                     scale=0.0, status=None) -> DecodeStepParams:
    B, H = query.shape[0], query.shape[1]
    if num_physical_blocks is None:
        num_physical_blocks = kv_pool.numel() // (2 * num_layers * block_size * num_kv_heads * head_dim)
    p = DecodeStepParams()
    p.query, p.key, p.value = query.data_ptr(), key.data_ptr(), value.data_ptr()
    p.qkv_dtype = _dtype_code(query)
    p.positions = positions.data_ptr()
    p.cos_sin = cos_sin.data_ptr() if cos_sin is not None else None
    p.max_position = cos_sin.shape[0] if cos_sin is not None else 0
    p.kv_pool, p.block_table = kv_pool.data_ptr(), block_table.data_ptr()
    p.num_physical_blocks = int(num_physical_blocks)
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim = B, H, num_kv_heads, head_dim
    p.block_size, p.num_layers, p.layer = block_size, num_layers, layer
    p.max_blocks_per_seq = block_table.shape[1]
    p.query_out = query_out.data_ptr() if query_out is not None else None
    if out is not None:
        p.out, p.out_dtype = out.data_ptr(), _dtype_code(out)
    p.scale = float(scale)
    p.status = status.data_ptr() if status is not None else None
    return p


@_streamed
def rope_append(query, key, value, positions, cos_sin, kv_pool, block_table, *, num_kv_heads, head_dim, block_size,
                num_layers=1, layer=0, query_out=None, status=None, stream=None):
    """RoPE on the new token's q/k and KV append (cottus_rope_append)."""
    for t, n in ((query, "query"), (key, "key"), (value, "value"), (kv_pool, "kv_pool")):
        _require(t, n)
    p = make_step_params(query, key, value, positions, cos_sin, kv_pool, block_table, num_kv_heads=num_kv_heads,
                         head_dim=head_dim, block_size=block_size, num_layers=num_layers, layer=layer,
                         query_out=query_out, status=status)
    check(lib().cottus_rope_append(C.byref(p), _stream(stream)))
    return query_out


@_streamed
def rope_append_decode(query, key, value, positions, cos_sin, kv_pool, block_table, *, num_kv_heads, head_dim,
                       block_size, num_layers=1, layer=0, out=None, out_dtype=None, query_out=None, scale=0.0,
                       status=None, stream=None, workspace_of=None):
    """RoPE + KV append + paged attention over positions+1 tokens (one kernel).  workspace_of: the DecodeBatch whose
    workspace serves the call; by default all calls on a device share one, and must not overlap on several streams."""
    for t, n in ((query, "query"), (key, "key"), (value, "value"), (kv_pool, "kv_pool")):
        _require(t, n)
    if out is None:
        out = torch.empty(query.shape, dtype=out_dtype or query.dtype, device=query.device)
    p = make_step_params(query, key, value, positions, cos_sin, kv_pool, block_table, num_kv_heads=num_kv_heads,
                         head_dim=head_dim, block_size=block_size, num_layers=num_layers, layer=layer,
                         query_out=query_out, out=out, scale=scale, status=status)
    need = lib().cottus_rope_append_decode_workspace_size(C.byref(p))
    if need:
        ws = workspace(need, query.device, stream=stream) if workspace_of is None else workspace_of.workspace(need, stream)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().cottus_rope_append_decode(C.byref(p), _stream(stream)))
    return out


@_streamed
def qkv_rope_append(x, weight, positions, cos_sin, kv_pool, block_table, *, num_heads, num_kv_heads, head_dim,
                    block_size, num_layers=1, layer=0, num_physical_blocks=None, query_out=None,
                    query_out_dtype=torch.float16, qkv_out=None, status=None, stream=None):
    """QKV projection + RoPE + KV append in one kernel (cottus_qkv_rope_append).
    x [B][hidden] fp16, weight [(H + 2 Hkv) D][hidden] fp16; returns the rotated query."""
    for t, n in ((x, "x"), (weight, "weight"), (kv_pool, "kv_pool")):
        _require(t, n)
    B, hidden = x.shape
    if num_physical_blocks is None:
        num_physical_blocks = kv_pool.numel() // (2 * num_layers * block_size * num_kv_heads * head_dim)
    if query_out is None:
        query_out = torch.empty((B, num_heads, head_dim), dtype=query_out_dtype, device=x.device)
    p = QkvParams()
    p.x, p.weight, p.hidden = x.data_ptr(), weight.data_ptr(), hidden
    p.positions, p.cos_sin, p.max_position = positions.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0]
    p.kv_pool, p.block_table, p.num_physical_blocks = kv_pool.data_ptr(), block_table.data_ptr(), int(num_physical_blocks)
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim = B, num_heads, num_kv_heads, head_dim
    p.block_size, p.num_layers, p.layer, p.max_blocks_per_seq = block_size, num_layers, layer, block_table.shape[1]
    p.query_out, p.query_out_dtype = query_out.data_ptr(), _dtype_code(query_out)
    p.qkv_out = qkv_out.data_ptr() if qkv_out is not None else None
    p.status = status.data_ptr() if status is not None else None
    need = lib().cottus_qkv_rope_append_workspace_size(C.byref(p))
    if need:
        ws = workspace(need, x.device, "proj", stream)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().cottus_qkv_rope_append(C.byref(p), _stream(stream)))
    return query_out


@_streamed
def o_proj_residual(x, weight, residual, *, out=None, out_dtype=torch.float32, status=None, stream=None):
    """Output projection + residual add (cottus_o_proj_residual):
    out = x . weight^T + residual.  x [B][in] fp16, weight [out][in] fp16,
    residual [B][out] fp32; out may be the residual tensor itself (fp32)."""
    for t, n in ((x, "x"), (weight, "weight"), (residual, "residual")):
        _require(t, n)
    B, fin = x.shape
    fout = weight.shape[0]
    if out is None:
        out = torch.empty((B, fout), dtype=out_dtype, device=x.device)
    p = OProjParams()
    p.x, p.weight, p.in_features, p.out_features, p.batch = x.data_ptr(), weight.data_ptr(), fin, fout, B
    p.residual, p.out, p.out_dtype = residual.data_ptr(), out.data_ptr(), _dtype_code(out)
    p.status = status.data_ptr() if status is not None else None
    need = lib().cottus_o_proj_residual_workspace_size(C.byref(p))
    if need:
        ws = workspace(need, x.device, "proj", stream)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().cottus_o_proj_residual(C.byref(p), _stream(stream)))
    return out


@_streamed
def attention_block(batch, x, w_qkv, w_o, residual, kv_pool, cos_sin, *, num_heads, num_kv_heads, head_dim,
                    num_layers=1, layer=0, query_out=None, att_out=None, status=None, stream=None):
    """The attention half of one decoder layer for the step tokens of a
    DecodeBatch (generic_transformer.cpp:169-327 per token), as three
    launches of this library: the QKV projection with RoPE and the KV append
    (cottus_qkv_rope_append), paged decode attention over the device block
    table with context = position + 1 (cottus_paged_decode), and the output
    projection added to the residual stream in place (cottus_o_proj_residual).

    x [n][hidden] fp16 (the normalised hidden state of each row's token, n =
    len(batch)), w_qkv [(H + 2 Hkv) D][hidden] fp16, w_o [hidden][H D] fp16,
    residual [n][hidden] fp32 (updated in place).  Returns the attention
    output [n][H D] fp16 (the O-projection's input)."""
    n = len(batch)
    if x.shape[0] != n or residual.shape[0] != n:
        raise ValueError(f"x and residual need one row per active sequence ({n})")
    nb = batch.num_blocks
    q = qkv_rope_append(x, w_qkv, batch.positions[:n], cos_sin, kv_pool, batch.block_table[:n], num_heads=num_heads,
                        num_kv_heads=num_kv_heads, head_dim=head_dim, block_size=batch.block_size,
                        num_layers=num_layers, layer=layer, num_physical_blocks=nb, query_out=query_out,
                        query_out_dtype=torch.float16, status=status, stream=stream)
    if att_out is None:
        att_out = torch.empty((n, num_heads, head_dim), dtype=torch.float16, device=x.device)
    paged_decode(q, kv_pool, batch.block_table[:n], batch.context_lens[:n], num_kv_heads=num_kv_heads,
                 head_dim=head_dim, block_size=batch.block_size, num_layers=num_layers, layer=layer, out=att_out,
                 status=status, num_physical_blocks=nb, stream=stream)
    att = att_out.view(n, num_heads * head_dim)
    o_proj_residual(att, w_o, residual, out=residual, status=status, stream=stream)
    return att


def _operand(t: torch.Tensor, name: str, shape, dtypes, device: int) -> int:
    """Checks one operand of the norm, 8-bit and sampling operators; its address."""
    if t.get_device() == device and t.dtype in dtypes and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.get_device() != device:
        raise ValueError(f"{name} is on cuda:{t.get_device()}, the current device is cuda:{device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _device() -> int:
    """The current device (torch.cuda.current_device without its check that CUDA is initialised, which a CUDA tensor
    implies: 0.1 of its 0.2 us)."""
    return torch._C._cuda_getDevice()


def _raw_stream(stream, device: int):
    """The stream's handle; of the current stream without building a Stream object (3.4 us of a 13 us call)."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device)
    if stream.device_index != device:  # (the default streams of all devices have one handle)
        raise ValueError(f"the stream is on cuda:{stream.device_index}, the current device is cuda:{device}")
    return stream.cuda_stream


_ONLY_F32, _ONLY_I32, _ONLY_FP8 = (torch.float32,), (torch.int32,), (_FP8,)


def _new(like: torch.Tensor, shape, dtype, stream) -> torch.Tensor:
    """A contiguous tensor of one or two dimensions (empty_strided parses its arguments in half the time of new_empty,
    1.8 us), of the memory pool of the stream that writes it: of another's it might hold what that one still reads."""
    strides = (shape[1], 1) if len(shape) == 2 else (1,)
    if stream is not None:
        with torch.cuda.stream(stream):
            return torch.empty_strided(shape, strides, dtype=dtype, device=like.device)
    return torch.empty_strided(shape, strides, dtype=dtype, device=like.device)


def _i32(n: int, name: str) -> int:
    """n as the C ABI's 32-bit sizes hold it (ctypes would drop the upper bits)."""
    if not 0 <= n < 1 << 31:
        raise ValueError(f"{name} is {n}, a 32-bit size")
    return n


def rms_norm(x, weight, *, eps=1e-5, residual=None, residual_out=None, out=None, out_dtype=None, scales=None,
             stream=None):
    """RMS norm with the residual's addition (cottus_rms_norm):
    h = x (+ residual), y = h / sqrt(mean(h^2) + eps) * weight.

    x [rows][hidden] fp32, fp16 or bf16; weight [hidden] fp32; residual [rows][hidden] fp32, replaced by h
    (or h goes to residual_out).  out_dtype defaults to x's.  Returns y, or, with out_dtype
    torch.float8_e4m3fn, (y, scales): scales [ceil(hidden / 128)][rows] fp32, y = values * their group's scale."""
    if x.dim() != 2:
        raise ValueError("x must be [rows][hidden]")
    dev = _device()
    shape = rows, hidden = x.shape
    p = RmsNormParams()
    p.x = _operand(x, "x", shape, _DT_WIDE, dev)
    p.weight = _operand(weight, "weight", (hidden,), _ONLY_F32, dev)
    if residual is not None:
        p.residual = _operand(residual, "residual", shape, _ONLY_F32, dev)
        p.residual_out = p.residual if residual_out is None else _operand(residual_out, "residual_out", x.shape,
                                                                          _ONLY_F32, dev)
    elif residual_out is not None:
        raise ValueError("residual_out goes with residual")
    if out is None:
        out = _new(x, (rows, hidden), out_dtype or x.dtype, stream)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise TypeError(f"out is {out.dtype}, out_dtype is {out_dtype}")
    fp8 = out.dtype == _FP8
    p.out = _operand(out, "out", shape, _ONLY_FP8 if fp8 else _DT_WIDE, dev)
    if fp8:
        if scales is None:
            scales = _new(x, ((hidden + 127) // 128, rows), torch.float32, stream)
        p.scales = _operand(scales, "scales", ((hidden + 127) // 128, rows), _ONLY_F32, dev)
    elif scales is not None:
        raise ValueError("scales go with a torch.float8_e4m3fn output")
    p.rows, p.hidden = rows, _i32(hidden, "hidden")
    p.x_dtype, p.out_dtype = _DT_WIDE[x.dtype], E4M3 if fp8 else _DT_WIDE[out.dtype]
    p.eps = eps
    check(lib().cottus_rms_norm(p, _raw_stream(stream, dev)))
    return (out, scales) if fp8 else out


def quantize_fp8(x, *, block_rows=1, out=None, scales=None, stream=None):
    """x [rows][cols] (fp32, fp16, bf16) in e4m3 with fp32 scales (cottus_quantize_fp8): (values, scales).
    block_rows 1: the activations of fp8_linear, one scale per row and 128 columns, [ceil(cols / 128)][rows];
    block_rows 128: its weight, one scale per 128 x 128 block, [ceil(rows / 128)][ceil(cols / 128)]."""
    if x.dim() != 2:
        raise ValueError("x must be [rows][cols]")
    dev = _device()
    rows, cols = x.shape
    p = QuantizeParams()
    p.x = _operand(x, "x", x.shape, _DT_WIDE, dev)
    if out is None:
        out = _new(x, (rows, cols), _FP8, stream)
    groups = (cols + 127) // 128
    shape = ((rows + 127) // 128, groups) if block_rows == 128 else (groups, rows)
    if scales is None:
        scales = _new(x, shape, torch.float32, stream)
    p.out = _operand(out, "out", x.shape, _ONLY_FP8, dev)
    p.scales = _operand(scales, "scales", shape, _ONLY_F32, dev)
    p.rows, p.cols, p.x_dtype, p.block_rows = rows, _i32(cols, "cols"), _DT_WIDE[x.dtype], _i32(block_rows, "block_rows")
    check(lib().cottus_quantize_fp8(p, _raw_stream(stream, dev)))
    return out, scales


def fp8_linear(x, x_scales, weight, weight_scales, *, residual=None, out=None, out_dtype=None, status=None, stream=None):
    """Block-scaled e4m3 product (cottus_fp8_linear): out = x . weight^T (+ residual), fp32 accumulation.
    x [rows][in] and x_scales from rms_norm or quantize_fp8; weight [out][in] and weight_scales from
    quantize_fp8(block_rows=128); residual [rows][out] fp32 (may be out itself where out is fp32).
    in a multiple of 16.  out_dtype: fp32, fp16 or bf16, by default out's, or fp16."""
    if x.dim() != 2 or weight.dim() != 2:
        raise ValueError("x must be [rows][in] and weight [out][in]")
    dev = _device()
    (rows, fin), fout = x.shape, weight.shape[0]
    groups = (fin + 127) // 128
    p = Fp8LinearParams()
    p.x = _operand(x, "x", x.shape, _ONLY_FP8, dev)
    p.x_scales = _operand(x_scales, "x_scales", (groups, rows), _ONLY_F32, dev)
    p.weight = _operand(weight, "weight", (fout, fin), _ONLY_FP8, dev)
    p.w_scales = _operand(weight_scales, "weight_scales", ((fout + 127) // 128, groups), _ONLY_F32, dev)
    if residual is not None:
        p.residual = _operand(residual, "residual", (rows, fout), _ONLY_F32, dev)
    if out is None:
        out = _new(x, (rows, fout), out_dtype or torch.float16, stream)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise TypeError(f"out is {out.dtype}, out_dtype is {out_dtype}")
    p.out = _operand(out, "out", (rows, fout), _DT_WIDE, dev)
    p.rows, p.out_features, p.in_features = _i32(rows, "rows"), _i32(fout, "out"), _i32(fin, "in")
    p.out_dtype = _DT_WIDE[out.dtype]
    if status is not None:
        p.status = _operand(status, "status", (1,), _ONLY_I32, dev)
    check(lib().cottus_fp8_linear(p, _raw_stream(stream, dev)))
    return out


def sample_tokens(logits, uniforms, *, temperature=None, top_k=None, top_p=None, min_p=None, out=None,
                  return_logprobs=False, logprobs=None, status=None, stream=None):
    """One token per row of logits [batch][vocab] (cottus_sample_tokens) from uniforms [batch] in [0, 1):
    temperature, then top-k, top-p and min-p, then the inverse of the running sum in index order.
    temperature, top_p and min_p are fp32 [batch], top_k int32 [batch]; None leaves a filter off
    (temperature: 1; a row with temperature 0 takes its largest logit).  Returns tokens int32 [batch] (-1 for a row
    without a finite logit), or (tokens, logprobs fp32 [batch]) with return_logprobs."""
    if logits.dim() != 2:
        raise ValueError("logits must be [batch][vocab]")
    dev = _device()
    batch, vocab = logits.shape
    row = (batch,)
    p = SampleParams()
    p.logits = _operand(logits, "logits", logits.shape, _DT_WIDE, dev)
    p.uniforms = _operand(uniforms, "uniforms", row, _ONLY_F32, dev)
    if temperature is not None:
        p.temperature = _operand(temperature, "temperature", row, _ONLY_F32, dev)
    if top_k is not None:
        p.top_k = _operand(top_k, "top_k", row, _ONLY_I32, dev)
    if top_p is not None:
        p.top_p = _operand(top_p, "top_p", row, _ONLY_F32, dev)
    if min_p is not None:
        p.min_p = _operand(min_p, "min_p", row, _ONLY_F32, dev)
    if out is None:
        out = _new(logits, row, torch.int32, stream)
    p.tokens = _operand(out, "out", row, _ONLY_I32, dev)
    if return_logprobs and logprobs is None:
        logprobs = _new(logits, row, torch.float32, stream)
    if logprobs is not None:
        p.logprobs = _operand(logprobs, "logprobs", row, _ONLY_F32, dev)
    if status is not None:
        p.status = _operand(status, "status", (1,), _ONLY_I32, dev)
    p.batch, p.vocab, p.dtype = _i32(batch, "batch"), _i32(vocab, "vocab"), _DT_WIDE[logits.dtype]
    check(lib().cottus_sample_tokens(p, _raw_stream(stream, dev)))
    return (out, logprobs) if return_logprobs else out


def attention_block_fp8(batch, residual, norm_weight, w_qkv, qkv_scales, w_o, o_scales, kv_pool, cos_sin, *, num_heads,
                        num_kv_heads, head_dim, eps=1e-5, num_layers=1, layer=0, status=None, stream=None):
    """attention_block on 8-bit weights, the norm in front included: for the step tokens of a DecodeBatch, from the
    residual stream back into it (generic_transformer.cpp:154-327 per token), as launches of this library: rms_norm to
    e4m3, the q, k and v projections (fp8_linear over row ranges of w_qkv), RoPE + append + paged decode
    (rope_append_decode), quantize_fp8 and the output projection added to the stream in place.

    residual [n][hidden] fp32 (updated), w_qkv [(H + 2 Hkv) D][hidden] and w_o [hidden][H D] e4m3 with the scales of
    quantize_fp8(block_rows=128); H D and Hkv D multiples of 128 (a range starts at a scale block).  Returns the
    attention output [n][H D] fp16.  Blocks of different batches may run on different streams at once."""
    if stream is not None:  # (what is allocated below belongs to the stream that writes it)
        with torch.cuda.stream(stream):
            return attention_block_fp8(batch, residual, norm_weight, w_qkv, qkv_scales, w_o, o_scales, kv_pool, cos_sin,
                                       num_heads=num_heads, num_kv_heads=num_kv_heads, head_dim=head_dim, eps=eps,
                                       num_layers=num_layers, layer=layer, status=status)
    n, qd, kd = len(batch), num_heads * head_dim, num_kv_heads * head_dim
    if residual.shape[0] != n:
        raise ValueError(f"residual needs one row per active sequence ({n})")
    if qd % 128 or kd % 128:
        raise ValueError("num_heads * head_dim and num_kv_heads * head_dim must be multiples of 128")
    if w_qkv.shape[0] != qd + 2 * kd:
        raise ValueError(f"w_qkv must have {qd + 2 * kd} rows")
    h, hs = rms_norm(residual, norm_weight, eps=eps, out_dtype=_FP8)
    qkv = []
    for r0, rows, heads in ((0, qd, num_heads), (qd, kd, num_kv_heads), (qd + kd, kd, num_kv_heads)):
        part = fp8_linear(h, hs, w_qkv[r0:r0 + rows], qkv_scales[r0 // 128:(r0 + rows) // 128], status=status)
        qkv.append(part.view(n, heads, head_dim))
    att = rope_append_decode(*qkv, batch.positions[:n], cos_sin, kv_pool, batch.block_table[:n],
                             num_kv_heads=num_kv_heads, head_dim=head_dim, block_size=batch.block_size,
                             num_layers=num_layers, layer=layer, status=status, workspace_of=batch).view(n, qd)
    a, a_scales = quantize_fp8(att)
    fp8_linear(a, a_scales, w_o, o_scales, residual=residual, out=residual, status=status)
    return att


def next_tokens(residual, norm_weight, w_head, head_scales, uniforms, *, eps=1e-5, temperature=None, top_k=None,
                top_p=None, min_p=None, logits=None, tokens=None, status=None, stream=None):
    """The end of a decode step (generic_transformer.cpp:369-370 and the argmax of engine.cpp:85-87), from the residual
    stream [n][hidden] fp32 to one token per row: the final rms_norm to e4m3, the vocabulary projection (fp8_linear,
    w_head [vocab][hidden] e4m3 with the scales of quantize_fp8(block_rows=128)) and sample_tokens.  Returns
    (tokens int32 [n], logits [n][vocab], fp32 unless a buffer of another type is given)."""
    h, hs = rms_norm(residual, norm_weight, eps=eps, out_dtype=_FP8, stream=stream)
    logits = fp8_linear(h, hs, w_head, head_scales, out=logits, out_dtype=None if logits is not None else torch.float32,
                        status=status, stream=stream)
    tokens = sample_tokens(logits, uniforms, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, out=tokens,
                           status=status, stream=stream)
    return tokens, logits


@_streamed
def paged_gather(kv_pool, block_table, context_lens, *, max_context, num_kv_heads, head_dim, block_size,
                 num_layers=1, layer=0, num_physical_blocks=None, status=None, k_out=None, v_out=None, stream=None):
    """Dense copy of the K and V rows named by the block table (bit-exact)."""
    B = block_table.shape[0]
    if num_physical_blocks is None:
        num_physical_blocks = kv_pool.numel() // (2 * num_layers * block_size * num_kv_heads * head_dim)
    if k_out is None:
        k_out = torch.zeros((B, max_context, num_kv_heads, head_dim), dtype=torch.uint16, device=kv_pool.device)
    if v_out is None:
        v_out = torch.zeros_like(k_out)
    check(lib().cottus_paged_gather(_ptr(k_out), _ptr(v_out), _ptr(kv_pool), _ptr(block_table), _ptr(context_lens),
                                    int(num_physical_blocks), B, max_context, num_kv_heads, head_dim, block_size,
                                    num_layers, layer, block_table.shape[1], _ptr(status), _stream(stream)))
    return k_out, v_out


class BlockAllocator:
    """The product's LIFO block pool (cottus_block_allocator_*), same
    semantics as the reference cottus::BlockAllocator."""

    def __init__(self, total_blocks: int, block_size: int):
        h = C.c_void_p()
        check(lib().cottus_block_allocator_create(total_blocks, block_size, C.byref(h)))
        self._h = h

    def allocate(self) -> int:
        bid = C.c_int32()
        check(lib().cottus_block_allocator_allocate(self._h, C.byref(bid)))
        return bid.value

    def free(self, block_id: int) -> None:
        check(lib().cottus_block_allocator_free(self._h, int(block_id)))

    def num_free(self) -> int:
        return int(lib().cottus_block_allocator_num_free(self._h))

    def total_blocks(self) -> int:
        return int(lib().cottus_block_allocator_total_blocks(self._h))

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            lib().cottus_block_allocator_destroy(h)
            self._h = None


class DecodeBatch:
    """Batched decode-step driver (cottus_decode_batch_*): the block
    bookkeeping of Engine::generate (engine.cpp:52-95) for many sequences,
    with the block table and positions resident on the device.

    `device` None keeps the host bookkeeping only.  Per step:
    ``begin_step()``, then per layer ``rope_append_decode(...)`` with
    ``block_table=self.block_table[:n]``, ``positions=self.positions[:n]``
    (n = len(self)), or ``attention_block(...)``, then ``end_step()``."""

    def __init__(self, num_blocks: int, block_size: int, max_batch: int, max_blocks_per_seq: int, device=None):
        self.block_table = self.positions = self.context_lens = None
        d = DecodeBatchDesc()
        d.num_blocks, d.block_size, d.max_batch, d.max_blocks_per_seq = num_blocks, block_size, max_batch, \
            max_blocks_per_seq
        if device is not None:
            self.block_table = torch.zeros((max_batch, max_blocks_per_seq), dtype=torch.int32, device=device)
            self.positions = torch.zeros(max_batch, dtype=torch.int32, device=device)
            self.context_lens = torch.zeros(max_batch, dtype=torch.int32, device=device)
            d.device_block_table, d.device_positions = self.block_table.data_ptr(), self.positions.data_ptr()
            d.device_context_lens = self.context_lens.data_ptr()
        h = C.c_void_p()
        check(lib().cottus_decode_batch_create(C.byref(d), C.byref(h)))
        self._h = h
        self.num_blocks, self.block_size = num_blocks, block_size
        self.max_batch, self.max_blocks_per_seq = max_batch, max_blocks_per_seq
        if device is not None:
            self._scratch = _Scratch(self.positions.device, cleared=True)
            # before any capture, and for all grouped-query shapes enough (2.5 MB for 8 query heads of 128 per kv head)
            self._scratch.get(4 << 20)
            if self.positions.is_cuda and not _capturing(self.positions.device):
                torch.cuda.current_stream(self.positions.device).synchronize()  # (the batch may be used on any stream)

    def workspace(self, nbytes: int, stream=None) -> torch.Tensor:
        """This batch's scratch buffer for the decode kernels (whose counter words are zero between calls)."""
        return self._scratch.get(nbytes, stream)

    def add(self, seq_id: int) -> int:
        row = C.c_int32()
        check(lib().cottus_decode_batch_add(self._h, int(seq_id), C.byref(row)))
        return row.value

    def release(self, seq_id: int) -> None:
        check(lib().cottus_decode_batch_release(self._h, int(seq_id)))

    def begin_step(self, stream=None) -> None:
        check(lib().cottus_decode_batch_begin_step(self._h, _stream(stream) if self.block_table is not None
                                                    else None))

    def end_step(self) -> None:
        check(lib().cottus_decode_batch_end_step(self._h))

    def __len__(self) -> int:
        return int(lib().cottus_decode_batch_size(self._h))

    def free_blocks(self) -> int:
        return int(lib().cottus_decode_batch_free_blocks(self._h))

    def rows(self) -> list:
        n = len(self)
        ids = (C.c_int64 * max(n, 1))()
        lib().cottus_decode_batch_rows(self._h, ids, n)
        return [int(ids[i]) for i in range(n)]

    def sequence(self, seq_id: int):
        """(row, next position, blocks) of an active sequence (host mirror)."""
        row, pos, nb = C.c_int32(), C.c_int32(), C.c_int32()
        check(lib().cottus_decode_batch_sequence(self._h, int(seq_id), C.byref(row), C.byref(pos), None, 0,
                                                 C.byref(nb)))
        blocks = (C.c_int32 * max(nb.value, 1))()
        check(lib().cottus_decode_batch_sequence(self._h, int(seq_id), None, None, blocks, nb.value, None))
        return row.value, pos.value, [int(blocks[i]) for i in range(nb.value)]

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            lib().cottus_decode_batch_destroy(h)
            self._h = None
