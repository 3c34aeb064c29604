"""krea2::ops::Ops::launch / launch_1d (src/ops/mod.rs:673-713) and the typed kernel calls.

Buffers are torch CUDA tensors (device memory and streams are torch's; the arithmetic is not):
each call passes raw device pointers through the C ABI of libkrea2_b200.so.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import kernels, shape
from ._lib import Binding, ConfigEntry, InvalidArgument, check, lib


def _stream_ptr(stream: Optional[torch.cuda.Stream]) -> int:
    return (stream or torch.cuda.current_stream()).cuda_stream


def _ptr(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise InvalidArgument("buffers must live on a CUDA device")
    if not t.is_contiguous():
        raise InvalidArgument("buffers must be contiguous")
    return t.data_ptr()


def _bytes(t: torch.Tensor) -> int:
    return t.numel() * t.element_size()


FLOAT_SCALARS = {"euler": "delta", "guidance": "scale"}


class Ops:
    """The generic dispatcher: kernel by name, config by key, scalars, buffers in binding order."""

    def launch(self, stream, name: str, config: kernels.Config, scalars: kernels.Scalars,
               bindings: Sequence[torch.Tensor], grid_x: int, grid_y: int, threads: int) -> None:
        kernels.grid(name, grid_x, grid_y)
        if scalars.floats and name in FLOAT_SCALARS:  # Scalars::float: the C ABI carries it as a config float
            config = {**config, FLOAT_SCALARS[name]: float(scalars.floats[0])}
        entries = (ConfigEntry * max(1, len(config)))()
        for i, (key, value) in enumerate(config.items()):
            entries[i].key = key.encode()
            if isinstance(value, float):
                entries[i].fvalue = value
            else:
                entries[i].value = int(value)
                entries[i].fvalue = float(value)
        indices = (ctypes.c_uint64 * max(1, len(scalars.indices)))(*scalars.indices)
        binds = (Binding * max(1, len(bindings)))()
        for i, t in enumerate(bindings):
            binds[i].ptr = _ptr(t)
            binds[i].bytes = _bytes(t)
        check(lib().krea2_launch(_stream_ptr(stream), name.encode(), entries, len(config), indices,
                                 len(scalars.indices), binds, len(bindings), grid_x, grid_y, threads))

    def launch_1d(self, stream, name, config, scalars, bindings, elements: int) -> None:
        """One 256-thread workgroup per 256 elements (src/ops/mod.rs:701-713)."""
        self.launch(stream, name, config, scalars, bindings, -(-elements // 256), 1, 256)


# ------------------------------------------------------------------ typed calls (C ABI order)
def prepare_norm_i8(h, norm_scale, mod_scale, mod_shift, q, q_scale, width, out_stride, eps=1e-5, stream=None):
    check(lib().krea2_prepare_norm_i8(_stream_ptr(stream), h.shape[0], _ptr(h), _ptr(norm_scale), _ptr(mod_scale),
                                      _ptr(mod_shift), _ptr(q), _ptr(q_scale), width, out_stride, eps))


def prepare_gated_i8(attn, gate, q, q_scale, width, out_stride, gate_stride, stream=None, tokens=None):
    tokens = attn.shape[0] if tokens is None else tokens
    check(lib().krea2_prepare_gated_i8(_stream_ptr(stream), tokens, _ptr(attn), gate.data_ptr(), _ptr(q),
                                       _ptr(q_scale), width, out_stride, gate_stride))


def prepare_plain_i8(h, q, q_scale, width, out_stride, stream=None):
    check(lib().krea2_prepare_plain_i8(_stream_ptr(stream), h.shape[0], _ptr(h), _ptr(q), _ptr(q_scale), width,
                                       out_stride))


def gemm_i8_256(m, a, w, scale, a_scale, c, k_size, k_stride, n_size, m_group=4, stream=None):
    check(lib().krea2_gemm_i8_256(_stream_ptr(stream), m, _ptr(a), _ptr(w), _ptr(scale), _ptr(a_scale), _ptr(c),
                                  k_size, k_stride, n_size, m_group))


def gemm_i8_resid_256(m, a, w, scale, a_scale, c, gate, k_size, k_stride, n_size, m_group=4, stream=None):
    check(lib().krea2_gemm_i8_resid_256(_stream_ptr(stream), m, _ptr(a), _ptr(w), _ptr(scale), _ptr(a_scale),
                                        _ptr(c), _ptr(gate), k_size, k_stride, n_size, m_group))


def gemm_i8_resid_256x256(m, a, w, scale, a_scale, c, gate, k_size, k_stride, n_size, m_group=4, schedule_rows=0,
                          stream=None):
    check(lib().krea2_gemm_i8_resid_256x256(_stream_ptr(stream), m, _ptr(a), _ptr(w), _ptr(scale), _ptr(a_scale),
                                            _ptr(c), _ptr(gate), k_size, k_stride, n_size, m_group,
                                            int(schedule_rows)))


def gemm_i8_swiglu_256(m, a, w, scale, a_scale, c, k_size, k_stride, n_size, m_group=4, stream=None):
    check(lib().krea2_gemm_i8_swiglu_256(_stream_ptr(stream), m, _ptr(a), _ptr(w), _ptr(scale), _ptr(a_scale),
                                         _ptr(c), k_size, k_stride, n_size, m_group))


def gemm_i8_swiglu_rotated_256(m, a, w, scale, a_scale, c, k_size, k_stride, n_size, m_group=4, stream=None):
    """gemm_i8_swiglu_256 whose epilogue also applies the first three rotation stages of prepare_plain_i8."""
    check(lib().krea2_gemm_i8_swiglu_rotated_256(_stream_ptr(stream), m, _ptr(a), _ptr(w), _ptr(scale), _ptr(a_scale),
                                                 _ptr(c), k_size, k_stride, n_size, m_group))


def prepare_rotated_i8(h, q, q_scale, width, out_stride, stream=None):
    """The rest of prepare_plain_i8 (last stage, row maximum, codes) on a row gemm_i8_swiglu_rotated_256 wrote."""
    check(lib().krea2_prepare_rotated_i8(_stream_ptr(stream), h.shape[0], _ptr(h), _ptr(q), _ptr(q_scale), width,
                                         out_stride))


def gemm_i8_rope_256(m, a, w, scale, a_scale, c, q_norm, k_norm, cos, sin, q_out, k_out, v_out, k_size, k_stride, n_size,
                     q_heads, kv_heads, eps=1e-5, m_group=4, stream=None):
    """gemm_i8_256 over q|k|v|gate columns whose epilogue also does rope_qknorm_f16's work: q, k normalised and
    rotated, v copied, only the gate columns written to `c`."""
    check(lib().krea2_gemm_i8_rope_256(_stream_ptr(stream), m, _ptr(a), _ptr(w), _ptr(scale), _ptr(a_scale), _ptr(c),
                                       _ptr(q_norm), _ptr(k_norm), _ptr(cos), _ptr(sin), _ptr(q_out), _ptr(k_out), _ptr(v_out),
                                       k_size, k_stride, n_size, m_group, q_heads, kv_heads, eps))


def gemm_i8_acc(m, a, w, acc, k_size, k_stride, n_size, stream=None):
    check(lib().krea2_gemm_i8_acc(_stream_ptr(stream), m, _ptr(a), _ptr(w), _ptr(acc), k_size, k_stride, n_size))


def lora_transport(src, dst, reverse: int, stream=None):
    check(lib().krea2_lora_transport(_stream_ptr(stream), src.numel(), _ptr(src), _ptr(dst), reverse))


class Quantized:
    """training::quantized::Quantized (src/training/quantized.rs:8-112): one W8A8 projection on
    bf16 tensors -- bf16 -> f16 transport, prepare_plain_i8, gemm_i8_256, f16 -> bf16."""

    def __init__(self, weight: torch.Tensor, scales: torch.Tensor, outputs: int, inputs: int):
        """`weight` int8 [outputs][inputs] and `scales` f32 [outputs], on the host or the device;
        rows are re-pitched to shape::gemm_pitch(inputs) as Quantized::load does (:34-47)."""
        if weight.dtype != torch.int8 or tuple(weight.shape) != (outputs, inputs) or scales.dtype != torch.float32 \
                or scales.numel() != outputs:
            raise InvalidArgument("invalid ConvRot projection")
        self.inputs, self.outputs = inputs, outputs
        self.pitch = shape.gemm_pitch(inputs)
        device = torch.device("cuda", torch.cuda.current_device())
        self.weight = torch.zeros((outputs, self.pitch), dtype=torch.int8, device=device)
        self.weight[:, :inputs] = weight.to(device)
        self.scales = scales.to(device).contiguous()

    def forward_fused(self, stream, x: torch.Tensor, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The same projection through krea2_quantized_forward: one C call, intermediates in a
        caller-owned workspace (allocated here when none is passed)."""
        if x.shape[-1] != self.inputs or x.dtype != torch.bfloat16:
            raise InvalidArgument("ConvRot projection dimensions")
        rows = x.shape[0]
        need = lib().krea2_quantized_workspace_bytes(rows, self.inputs, self.outputs)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        out = torch.empty((rows, self.outputs), dtype=torch.bfloat16, device=x.device)
        check(lib().krea2_quantized_forward(_stream_ptr(stream), rows, _ptr(x), _ptr(self.weight), _ptr(self.scales),
                                            _ptr(out), self.inputs, self.outputs, _ptr(workspace), _bytes(workspace)))
        return out

    def forward(self, ops: Ops, stream, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.inputs or x.dtype != torch.bfloat16:
            raise InvalidArgument("ConvRot projection dimensions")
        rows = x.shape[0]
        dev = x.device
        transport = torch.empty((rows, self.inputs), dtype=torch.float16, device=dev)
        quantized = torch.empty((rows, self.pitch), dtype=torch.int8, device=dev)
        scales = torch.empty((rows,), dtype=torch.float32, device=dev)
        out_f16 = torch.empty((rows, self.outputs), dtype=torch.float16, device=dev)
        out = torch.empty((rows, self.outputs), dtype=torch.bfloat16, device=dev)
        one = kernels.Scalars()
        ops.launch_1d(stream, "lora_transport", kernels.config([("reverse", 1)]), one.index(x.numel()),
                      [x, transport], x.numel())
        ops.launch(stream, "prepare_plain_i8", kernels.config([("width", self.inputs), ("out_stride", self.pitch)]),
                   one.index(rows), [transport, quantized, scales], rows, 1, 256)
        ops.launch(stream, "gemm_i8_256",
                   kernels.config([("k_size", self.inputs), ("k_stride", self.pitch), ("n_size", self.outputs),
                                   ("m_group", shape.gemm_m_group())]),
                   one.index(rows), [quantized, self.weight, self.scales, scales, out_f16], self.outputs // 128,
                   shape.gemm_grid_rows(rows), 256)
        ops.launch_1d(stream, "lora_transport", kernels.config([("reverse", 2)]), one.index(out.numel()),
                      [out_f16, out], out.numel())
        return out


# ------------------------------------------------------------------ the rest of a block
def rope_qknorm_f16(qkv, q_scale, k_scale, cos, sin, q_out, k_out, v_out, row_stride, q_heads, kv_heads, k_offset,
                    eps=1e-5, stream=None, tokens=None):
    tokens = q_out.shape[0] if tokens is None else tokens
    check(lib().krea2_rope_qknorm_f16(_stream_ptr(stream), tokens, qkv.data_ptr(), _ptr(q_scale), _ptr(k_scale), _ptr(cos),
                                      _ptr(sin), _ptr(q_out), _ptr(k_out), _ptr(v_out), row_stride, q_heads, kv_heads,
                                      k_offset, eps))


def v_transpose(x, out, width, row_capacity, stream=None, rows=None):
    rows = x.shape[0] if rows is None else rows
    check(lib().krea2_v_transpose(_stream_ptr(stream), rows, _ptr(x), _ptr(out), width, row_capacity))


def attention_gqa(tokens, kv_heads, q, k, v_transposed, out, q_stride, kv_stride, out_stride, token_capacity, scale,
                  stream=None, q32=False):
    fn = lib().krea2_attention_gqa_lds_f16_wmma_q32 if q32 else lib().krea2_attention_gqa_lds_f16_wmma
    check(fn(_stream_ptr(stream), tokens, kv_heads, _ptr(q), _ptr(k), _ptr(v_transposed), _ptr(out), q_stride, kv_stride,
             out_stride, token_capacity, scale))


def attention_gqa_rows(q_rows, tokens, kv_heads, q, k, v_transposed, out, q_stride, kv_stride, out_stride, token_capacity,
                       scale, stream=None):
    """`q_rows` query rows (q and out hold just those) against all `tokens` keys and values."""
    check(lib().krea2_attention_gqa_f16_rows(_stream_ptr(stream), q_rows, tokens, kv_heads, _ptr(q), _ptr(k),
                                             _ptr(v_transposed), _ptr(out), q_stride, kv_stride, out_stride,
                                             token_capacity, scale))


def rope_qknorm_f16_sharded(tokens, qkv, q_scale, k_scale, cos, sin, q_out, row_stride, q_heads, kv_heads, k_offset,
                            shard, eps=1e-5, stream=None):
    """QK-norm + RoPE of this device's rows; K and V rows go to every device's full-length tensors (`shard`:
    a `_lib.RowShard`)."""
    check(lib().krea2_rope_qknorm_f16_sharded(_stream_ptr(stream), tokens, qkv.data_ptr(), _ptr(q_scale), _ptr(k_scale),
                                              _ptr(cos), _ptr(sin), _ptr(q_out), row_stride, q_heads, kv_heads, k_offset,
                                              eps, ctypes.byref(shard)))


def shard_signal(shard, stream=None):
    check(lib().krea2_shard_signal(_stream_ptr(stream), ctypes.byref(shard)))


# ------------------------------------------------------------------ around the block chain
def modulation(vector, tables, out, stream=None):
    """Models::modulation (src/models/graph.rs:405-425): `out` f32 = bf16(vector[i % len] + tables[i])."""
    if out.numel() != tables.numel():
        raise InvalidArgument("modulation dimensions")
    check(lib().krea2_modulation(_stream_ptr(stream), tables.numel(), _ptr(vector), _ptr(tables), _ptr(out),
                                 vector.numel()))


def euler_step(sample, velocity, delta, stream=None):
    """Ops::euler_step (src/ops/mod.rs:373-390): `sample += delta * velocity` in place with the sampler's
    bf16 rounding at the delta, the product and the sum."""
    if tuple(sample.shape) != tuple(velocity.shape):
        raise InvalidArgument("scheduler tensor dimensions")
    check(lib().krea2_euler(_stream_ptr(stream), sample.numel(), float(delta), _ptr(sample), _ptr(velocity)))


def guidance(cond, uncond, scale, stream=None):
    """Ops::guidance (src/ops/mod.rs:392-410): `cond += scale * (cond - uncond)` in place, bf16 at each step."""
    if tuple(cond.shape) != tuple(uncond.shape):
        raise InvalidArgument("guidance tensor dimensions")
    check(lib().krea2_guidance(_stream_ptr(stream), cond.numel(), float(scale), _ptr(cond), _ptr(uncond)))


# ------------------------------------------------------------------ e4m3 projections, rotary positions, cross attention
# New with this library.  Rows may have any pitch the C ABI takes (a slice of a wider tensor is fine); a call runs on the
# tensors' device, on `stream` or that device's current stream.
KINDS = {torch.float16: 0, torch.bfloat16: 1}
GROUP = 128  # channels under one scale
ROTARY_LAYOUTS = {"interleaved": 0, "half": 1}
ROTARY_SCALINGS = {"none": 0, "linear": 1, "base": 2, "parts": 3}


def _groups(width: int) -> int:
    return -(-width // GROUP)


def _kind(name, t: torch.Tensor) -> int:
    kind = KINDS.get(t.dtype)
    if kind is None:
        raise InvalidArgument(f"{name}: {t.dtype} is neither float16 nor bfloat16")
    return kind


def _dims(name, t: torch.Tensor, rank: int):
    if t.dim() != rank:
        raise InvalidArgument(f"{name}: a tensor of {rank} dimensions is needed, got {tuple(t.shape)}")
    return t.shape


def _rows(name, what, t, shape, dtype, device, inner, lead=1) -> int:
    """Elements from one row of `t` to the next, where it has that shape and type, lies on that device and its dimensions
    after the first `lead` in one piece of `inner` elements.  A lone row's stride carries no meaning: it counts as `inner`."""
    if t.dtype is not dtype or t.shape != shape:
        raise InvalidArgument(f"{name}: {what} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise InvalidArgument(f"{name}: {what} is on {t.device}: buffers must share one CUDA device")
    if t.is_contiguous():
        return inner
    size, strides = 1, t.stride()
    for i in range(len(shape) - 1, lead - 1, -1):
        if shape[i] != 1 and strides[i] != size:
            raise InvalidArgument(f"{name}: the rows of {what} must be contiguous")
        size *= shape[i]
    return strides[lead - 1] if shape[lead - 1] > 1 else inner


def _pitch(t: torch.Tensor, stride: int) -> int:
    """The row pitch of codes: that of a lone row, whatever it says, is taken as the next multiple of 16."""
    return stride if t.shape[0] > 1 else _padded(stride)


def _padded(stride: int) -> int:
    return -(-stride // 16) * 16


# The current stream of a device as a pointer, and the current device once there are CUDA tensors; torch.cuda.current_stream()
# takes 3 us of a small call's 12.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _run_on(name, device: torch.device, stream, fn, *args) -> None:
    if device.type != "cuda":
        raise InvalidArgument(f"{name}: buffers must live on a CUDA device")
    index = device.index
    if stream is not None and stream.device != device:
        raise InvalidArgument(f"{name}: the stream belongs to {stream.device}, the buffers to {device}")
    pointer = stream.cuda_stream if stream is not None else _raw_stream(index)
    if index == _current_device():
        status = fn(pointer, *args)
    else:
        with torch.cuda.device(index):
            status = fn(pointer, *args)
    if status:
        check(status)


def prepare_norm_fp8(x, weight, q, q_scale, residual=None, sum_out=None, eps=1e-5, weight_offset=0.0, stream=None):
    """RMS norm of x [tokens][width] (after x + residual, which `sum_out` receives, if there is one) times
    (weight_offset + weight), as e4m3 codes q with q_scale f32 [tokens][ceil(width/128)]."""
    name, device, shape, dtype = "prepare_norm_fp8", x.device, x.shape, x.dtype
    kind, (tokens, width) = _kind(name, x), _dims(name, x, 2)
    x_stride = _rows(name, "x", x, shape, dtype, device, width)
    q_stride = _pitch(q, _rows(name, "q", q, shape, torch.float8_e4m3fn, device, width))
    _rows(name, "q_scale", q_scale, (tokens, -(-width // GROUP)), torch.float32, device, width)
    residual_ptr = weight_ptr = sum_ptr = None
    residual_stride = sum_stride = 0
    if residual is not None:
        residual_stride, residual_ptr = _rows(name, "residual", residual, shape, dtype, device, width), residual.data_ptr()
    if sum_out is not None:
        sum_stride, sum_ptr = _rows(name, "sum_out", sum_out, shape, dtype, device, width), sum_out.data_ptr()
    if weight is not None:
        if weight.dtype is not torch.float32 or weight.numel() != width or weight.device != device:
            raise InvalidArgument(f"{name}: weight must be float32 [{width}] on {device}")
        weight_ptr = _ptr(weight)
    _run_on(name, device, stream, lib().krea2_prepare_norm_fp8, tokens, x.data_ptr(), residual_ptr, weight_ptr, sum_ptr, q.data_ptr(), _ptr(q_scale),
            width, x_stride, residual_stride, sum_stride, q_stride, eps, weight_offset, kind)


def prepare_plain_fp8(x, q, q_scale, stream=None):
    """e4m3 codes of x [tokens][width] with one scale per 128 channels (prepare_norm_fp8 without the norm)."""
    name, device, shape = "prepare_plain_fp8", x.device, x.shape
    kind, (tokens, width) = _kind(name, x), _dims(name, x, 2)
    x_stride = _rows(name, "x", x, shape, x.dtype, device, width)
    q_stride = _pitch(q, _rows(name, "q", q, shape, torch.float8_e4m3fn, device, width))
    _rows(name, "q_scale", q_scale, (tokens, -(-width // GROUP)), torch.float32, device, width)
    _run_on(name, device, stream, lib().krea2_prepare_plain_fp8, tokens, x.data_ptr(), q.data_ptr(), _ptr(q_scale), width, x_stride, q_stride, kind)


def gemm_fp8_128(a, a_scale, w, w_scale, c, stream=None):
    """c [m][n] (f16 or bf16) = a [m][k] times w [n][k] transposed, e4m3 codes under a_scale f32 [m][ceil(k/128)] and
    w_scale f32 [ceil(n/128)][ceil(k/128)]."""
    name, device = "gemm_fp8_128", a.device
    kind, (m, k), (n, _) = _kind(name, c), _dims(name, a, 2), _dims(name, w, 2)
    groups = -(-k // GROUP)
    a_stride = _pitch(a, _rows(name, "a", a, a.shape, torch.float8_e4m3fn, device, k))
    w_stride = _pitch(w, _rows(name, "w", w, (n, k), torch.float8_e4m3fn, device, k))
    _rows(name, "a_scale", a_scale, (m, groups), torch.float32, device, groups)
    _rows(name, "w_scale", w_scale, (-(-n // GROUP), groups), torch.float32, device, groups)
    c_stride = _rows(name, "c", c, (m, n), c.dtype, device, n)
    _run_on(name, device, stream, lib().krea2_gemm_fp8_128, m, a.data_ptr(), w.data_ptr(), _ptr(w_scale), _ptr(a_scale), c.data_ptr(), k, a_stride,
            w_stride, n, c_stride, kind)


class QuantizedFp8:
    """One projection on f16 or bf16 rows through e4m3 codes (the e4m3 sibling of Quantized): prepare_plain_fp8, or
    prepare_norm_fp8 where a norm precedes it, then gemm_fp8_128."""

    def __init__(self, weight: torch.Tensor):
        """`weight` [outputs][inputs] in a floating type on the device that the calls will run on; kept as e4m3 codes with
        one scale per 128 x 128 block."""
        if weight.dim() != 2 or not weight.is_floating_point() or not weight.is_cuda or 0 in weight.shape:
            raise InvalidArgument("an e4m3 projection takes a floating CUDA weight [outputs][inputs]")
        self.outputs, self.inputs = weight.shape
        weight = weight.detach()
        rows, columns = _groups(self.outputs), _groups(self.inputs)
        blocks = torch.zeros((rows * GROUP, columns * GROUP), dtype=torch.float32, device=weight.device)
        blocks[: self.outputs, : self.inputs] = weight
        blocks = blocks.view(rows, GROUP, columns, GROUP)
        self.scales = (blocks.abs().amax((1, 3)) / 448.0).clamp_min_(2.0 ** -126)
        codes = (blocks / self.scales[:, None, :, None]).clamp_(-448.0, 448.0).view(rows * GROUP, columns * GROUP)
        pitch = _padded(self.inputs)
        codes = codes[: self.outputs, : pitch].to(torch.float8_e4m3fn).view(torch.uint8).contiguous()
        self.weight = codes.view(torch.float8_e4m3fn)[:, : self.inputs]

    def buffers(self, rows: int):
        """Codes and scales of `rows` input rows, for a caller that keeps them between calls."""
        device = self.weight.device
        q = torch.empty((rows, _padded(self.inputs)), dtype=torch.float8_e4m3fn, device=device)[:, : self.inputs]
        return q, torch.empty((rows, _groups(self.inputs)), dtype=torch.float32, device=device)

    def forward(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, buffers=None, stream=None) -> torch.Tensor:
        """x [rows][inputs] -> [rows][outputs] in x's type."""
        return self._forward(x, out, buffers, stream, lambda q, s: prepare_plain_fp8(x, q, s, stream=stream))

    def forward_norm(self, x: torch.Tensor, norm_weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None,
                     sum_out: Optional[torch.Tensor] = None, eps: float = 1e-5, weight_offset: float = 0.0,
                     out: Optional[torch.Tensor] = None, buffers=None, stream=None) -> torch.Tensor:
        """The projection of the RMS norm of x (+ residual, whose sum `sum_out` receives)."""
        return self._forward(x, out, buffers, stream, lambda q, s: prepare_norm_fp8(
            x, norm_weight, q, s, residual=residual, sum_out=sum_out, eps=eps, weight_offset=weight_offset, stream=stream))

    def _forward(self, x, out, buffers, stream, prepare):
        if x.dim() != 2 or x.shape[1] != self.inputs:
            raise InvalidArgument("e4m3 projection dimensions")
        # What is not given is allocated on the stream that uses it, so that the allocator reuses it in that stream's order.
        with torch.cuda.stream(stream):
            q, scale = buffers or self.buffers(x.shape[0])
            if out is None:
                out = torch.empty((x.shape[0], self.outputs), dtype=x.dtype, device=x.device)
        prepare(q, scale)
        gemm_fp8_128(q, scale, self.weight, self.scales, out, stream=stream)
        return out


def rotary_frequencies(rotary_dim, base=10000.0, scaling="none", factor=1.0, trained=0.0, slow=1.0, fast=32.0, device=None):
    """(frequencies f64 [rotary_dim / 2] on `device`, magnitude) for ops.rotary; `scaling` "none", "linear", "base" or
    "parts" for contexts `factor` times the `trained` length."""
    if scaling not in ROTARY_SCALINGS:
        raise InvalidArgument(f"rotary_frequencies: scaling is one of {', '.join(ROTARY_SCALINGS)}")
    out = torch.empty(max(0, int(rotary_dim)) // 2, dtype=torch.float64)
    magnitude = ctypes.c_float()
    check(lib().krea2_rotary_frequencies(max(0, int(rotary_dim)), base, ROTARY_SCALINGS[scaling], factor, trained, slow, fast, out.data_ptr(),
                                         ctypes.byref(magnitude)))
    return out.to(device or "cuda"), magnitude.value


def rotary(q, k, q_out, k_out, frequencies, positions=None, magnitude=1.0, layout="interleaved", inverse=False, stream=None):
    """Turns q [tokens][q_heads][head_dim] and k [tokens][kv_heads][head_dim] (or None) by positions * frequencies into
    q_out and k_out, which may be q and k; the first 2 * len(frequencies) channels of a head take part.  inverse=True is
    the gradient's way back."""
    name, device, shape, dtype = "rotary", q.device, q.shape, q.dtype
    kind, (tokens, q_heads, head_dim) = _kind(name, q), _dims(name, q, 3)
    row = q_heads * head_dim
    q_stride, q_out_stride = _rows(name, "q", q, shape, dtype, device, row), _rows(name, "q_out", q_out, shape, dtype, device, row)
    kv_heads = k_stride = k_out_stride = 0
    k_ptr = k_out_ptr = positions_ptr = None
    if (k is None) != (k_out is None):
        raise InvalidArgument(f"{name}: k and k_out go together")
    if k is not None:
        kv_heads = _dims(name, k, 3)[1]
        shape, row = (tokens, kv_heads, head_dim), kv_heads * head_dim
        k_stride, k_out_stride = _rows(name, "k", k, shape, dtype, device, row), _rows(name, "k_out", k_out, shape, dtype, device, row)
        k_ptr, k_out_ptr = k.data_ptr(), k_out.data_ptr()
    if layout not in ROTARY_LAYOUTS:
        raise InvalidArgument(f"{name}: layout is one of {', '.join(ROTARY_LAYOUTS)}")
    if frequencies.dtype is not torch.float64 or frequencies.device != device:
        raise InvalidArgument(f"{name}: frequencies must be float64 on {device}")
    if positions is not None:
        if positions.dtype is not torch.int32 or positions.numel() != tokens or positions.device != device:
            raise InvalidArgument(f"{name}: positions must be int32 [{tokens}] on {device}")
        positions_ptr = _ptr(positions)
    _run_on(name, device, stream, lib().krea2_rotary, tokens, q.data_ptr(), k_ptr, positions_ptr, _ptr(frequencies), q_out.data_ptr(), k_out_ptr,
            q_heads, kv_heads, head_dim, 2 * frequencies.numel(), q_stride, k_stride, q_out_stride, k_out_stride, magnitude, ROTARY_LAYOUTS[layout],
            1 if inverse else 0, kind)


def cross_attention(q, k, v, out, kv_lengths=None, key_mask=None, scale=None, stream=None):
    """Attention of q [batch][q_len][q_heads][head_dim] to an encoder's k, v [batch][kv_len][kv_heads][head_dim], written
    to `out` (shaped like q).  kv_lengths int32 [batch] and key_mask bool or uint8 [batch][kv_len] say which keys count
    (both: those that both name); a query without one gets zeros.  scale defaults to head_dim ** -0.5."""
    name, device, shape, dtype = "cross_attention", q.device, q.shape, q.dtype
    kind, (batch, q_len, q_heads, head_dim), (_, kv_len, kv_heads, _) = _kind(name, q), _dims(name, q, 4), _dims(name, k, 4)

    def strides(what, t, shape, row):
        """(batch stride, row stride)"""
        stride = _rows(name, what, t, shape, dtype, device, row, 2)
        if batch == 1 or t.is_contiguous():
            return shape[1] * stride, stride
        return t.stride()[0], stride

    q_row, kv_row, kv_shape = q_heads * head_dim, kv_heads * head_dim, (batch, kv_len, kv_heads, head_dim)
    q_strides, out_strides = strides("q", q, shape, q_row), strides("out", out, shape, q_row)
    k_strides, v_strides = strides("k", k, kv_shape, kv_row), strides("v", v, kv_shape, kv_row)
    lengths_ptr = mask_ptr = None
    mask_stride = 0
    if kv_lengths is not None:
        if kv_lengths.dtype is not torch.int32 or kv_lengths.numel() != batch or kv_lengths.device != device:
            raise InvalidArgument(f"{name}: kv_lengths must be int32 [{batch}] on {device}")
        lengths_ptr = _ptr(kv_lengths)
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8):
            raise InvalidArgument(f"{name}: key_mask must be bool or uint8")
        mask_stride, mask_ptr = _rows(name, "key_mask", key_mask, (batch, kv_len), key_mask.dtype, device, kv_len), key_mask.data_ptr()
    _run_on(name, device, stream, lib().krea2_cross_attention, batch, q_len, kv_len, q.data_ptr(), k.data_ptr(), v.data_ptr(), lengths_ptr, mask_ptr,
            out.data_ptr(), q_heads, kv_heads, head_dim, *q_strides, *k_strides, *v_strides, *out_strides, mask_stride,
            max(1, head_dim) ** -0.5 if scale is None else scale, kind)
