"""Ready-made ops on top of ``torch.ops.sideaware.elementwise``: RoPE (llm.c formula), bf16
scale+bias and fill.  Each builds its op header once per shape (``headers.py``), registers it with
the library and launches through the same custom op a user-written header would use.

The frequency table is an *input*: build it on the host with ``freqs_cis_table`` (the llm.c
formula, ``example_llmc_rope.cu:19-52``) or bring your own, as (T, head_dim) fp32 with cos at
even and sin at odd columns.
"""
from __future__ import annotations

import ctypes
import math
import os
import struct
from typing import Dict, Optional, Tuple

import torch

from . import headers, wrapper

_kernel_ids: Dict[Tuple, int] = {}
_CHECK_POSITION_VALUES = os.environ.get("SIDEAWARE_CHECK_POSITIONS") == "1"

_HEADER_BUILDERS = {
    "rope": headers.rope_header,
    "rope_half": headers.rope_half_header,
    "scale_bias_bf16": headers.scale_bias_bf16_header,
    "mxfp8_quantize": headers.mxfp8_quantize_header,
    "mxfp8_dequantize": headers.mxfp8_dequantize_header,
    "fill": headers.fill_header,
    "rope_axes": headers.rope_axes_header,
    "dropout": headers.dropout_header,
}


@torch.compiler.assume_constant_result
def _kernel(builder: str, args: Tuple = (), kwargs: Tuple = ()) -> int:
    """The kernel id of the op whose header is ``_HEADER_BUILDERS[builder](*args, **dict(kwargs))``,
    registering it on first use.  Everything it takes is a constant (strings, ints, bools), so a
    tracer evaluates the call once, while it traces, and keeps the id as a constant of the graph:
    an op whose first use falls inside ``torch.compile(fullgraph=True)`` needs no eager warm-up."""
    key = (builder, args, kwargs)
    kid = _kernel_ids.get(key)
    if kid is None:
        kid = wrapper.sideaware_create_kernel(_HEADER_BUILDERS[builder](*args, **dict(kwargs)))
        _kernel_ids[key] = kid
    return kid


def _elementwise(*args) -> None:
    """The elementwise op.  Eager code goes straight to the op's implementation, the function
    ``torch.ops.sideaware.elementwise`` dispatches to, and saves the dispatcher's per-call cost
    (about a microsecond of a small launch); under ``torch.compile`` the call goes through the
    registered op, which the tracer keeps as one opaque node."""
    if torch.compiler.is_compiling():
        torch.ops.sideaware.elementwise(*args)
    else:
        wrapper.sideaware_elementwise(*args)


def freqs_cis_table(head_dim: int, end: int, theta: float, use_scaled: bool = False) -> torch.Tensor:
    """(end, head_dim) fp32 table on the host: [t, 2i] = cos(t*f_i), [t, 2i+1] = sin(t*f_i),
    f_i = theta^(-2i/head_dim) in fp32, optionally with the Llama-3.1 wavelength rescaling
    (``example_llmc_rope.cu:25-43``).  Built with torch CPU ops in fp32."""
    i = torch.arange(head_dim // 2, dtype=torch.float32)
    freq = 1.0 / torch.pow(torch.tensor(theta, dtype=torch.float32), (2 * i) / head_dim)
    if use_scaled:
        scale_factor, low_factor, high_factor, old_len = 8.0, 1.0, 4.0, 8192.0
        wavelen = (2.0 * math.pi / freq.double()).float()
        smooth = (old_len / wavelen - low_factor) / (high_factor - low_factor)
        blended = (1.0 - smooth) * freq / scale_factor + smooth * freq
        freq = torch.where(wavelen < old_len / high_factor, freq,
                           torch.where(wavelen > old_len / low_factor, freq / scale_factor, blended))
    angle = torch.arange(end, dtype=torch.float32)[:, None] * freq[None, :]
    table = torch.empty(end, head_dim, dtype=torch.float32)
    table[:, 0::2] = torch.cos(angle)
    table[:, 1::2] = torch.sin(angle)
    return table


_ROPE_DTYPES = {torch.float32: "fp32", torch.bfloat16: "bf16", torch.float16: "fp16"}


def _check_positions(positions: torch.Tensor, tokens: int, x: torch.Tensor, rows: int) -> None:
    """The kernel reads table row ``positions[token]`` without a bound (a check per element would
    cost more than the op): shape, type and device are checked here, and with
    ``SIDEAWARE_CHECK_POSITIONS=1`` in the environment the values too (a device round trip)."""
    assert positions.dtype == torch.int32 and positions.is_cuda and positions.is_contiguous(), \
        "positions are a contiguous int32 device tensor"
    assert positions.device == x.device, "positions live on the activations' device"
    assert positions.numel() == tokens, "one position per token of the flattened (B, T) axes"
    if _CHECK_POSITION_VALUES and tokens:
        lo, hi = int(positions.min()), int(positions.max())
        assert 0 <= lo and hi < rows, "positions must lie in [0, %d): got %d .. %d" % (rows, lo, hi)


def _rope(x: torch.Tensor, freqs: torch.Tensor, out: Optional[torch.Tensor], n_q: int, n_kv: int,
          layout: str, backward: bool, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    assert x.dim() == 4, "activations are (B, T, heads, head_dim)"
    B, T, heads, head_dim = x.shape
    if layout == "qkv":
        assert heads == n_q + 2 * n_kv, "packed QKV needs n_q + 2*n_kv heads"
    else:
        n_q, n_kv = heads, 0
    dtype = _ROPE_DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError("RoPE storage is float32, bfloat16 or float16")
    if positions is None:
        assert freqs.dtype == torch.float32 and freqs.shape == (T, head_dim)
    else:
        assert layout == "heads", "positions go with separate q / k tensors"
        assert freqs.dtype == torch.float32 and freqs.dim() == 2 and freqs.shape[1] == head_dim
        _check_positions(positions, B * T, x, freqs.shape[0])
        T = 0                                   # the sequence length is not part of the compiled text
    if out is None:
        out = x
    else:
        assert out.shape == x.shape and out.dtype == x.dtype
        if layout == "qkv" and out.data_ptr() != x.data_ptr():
            # value heads are skipped by the kernel (neither read nor written): out of place they
            # have to be carried over by a copy first
            torch.ops.sideaware.memcpy(out, x)
    kid = _kernel("rope", (max(T, 1), n_q, n_kv, head_dim, dtype, layout, backward),
                  (("positions", positions is not None),))
    _elementwise(kid, out, None, None, None, x, freqs, None, None, positions, 0, 0, 0)
    return out


def rope_forward_qkv(x, freqs, n_q: int, n_kv: int, out=None):
    """Packed (B, T, n_q + 2*n_kv, head_dim): rotates q and k heads, leaves v heads alone.
    In place unless ``out`` is given."""
    return _rope(x, freqs, out, n_q, n_kv, "qkv", False)


def rope_backward_qkv(dout, freqs, n_q: int, n_kv: int, out=None):
    return _rope(dout, freqs, out, n_q, n_kv, "qkv", True)


def rope_forward_heads(x, freqs, out=None, positions=None):
    """(B, T, heads, head_dim), every head rotated: one call per separate q or k tensor.
    ``positions``: an int32 device tensor with one table row number per token of the flattened
    (B, T) axes, for decoding steps and packed sequences (``freqs`` then has a row for every
    position that occurs); without it token t of every sequence uses row t."""
    return _rope(x, freqs, out, 0, 0, "heads", False, positions)


def rope_backward_heads(dout, freqs, out=None, positions=None):
    return _rope(dout, freqs, out, 0, 0, "heads", True, positions)


class _Segment(ctypes.Structure):
    """``sideaware_segment`` of include/sideaware.h."""
    _fields_ = [("num_bytes", ctypes.c_size_t), ("out", ctypes.c_void_p * 4), ("inp", ctypes.c_void_p * 4),
                ("sideband_memory", ctypes.c_void_p), ("sideband_value", ctypes.c_int)]


# The same layout, filled in one step (field by field costs a small launch several times its C call).  The sideband value
# goes in as the word its low 32 bits are, as ctypes passes it in a single launch: a bit pattern of 2^31 or more is one too.
_SEGMENT = struct.Struct("=Q4Q4QQI4x")
_WORD = 0xFFFFFFFF
assert _SEGMENT.size == ctypes.sizeof(_Segment)


def elementwise_batch(kernel_id: int, segments) -> None:
    """One launch over several arrays of the same op.  ``segments`` is a sequence of
    ``(num_bytes, outs, ins, sideband_tensor_or_None, sideband_value)`` with ``outs`` / ``ins``
    sequences of up to four tensors (or None)."""
    packed, first = [], None
    for num_bytes, outs, ins, sideband, value in segments:
        out, inp = [0] * 4, [0] * 4
        for i, t in enumerate(outs):
            out[i] = wrapper._check(t, "out%d" % i)
            first = t if first is None else first
        for i, t in enumerate(ins):
            inp[i] = wrapper._check(t, "in%d" % i)
            first = t if first is None else first
        packed.append(_SEGMENT.pack(num_bytes, *out, *inp, sideband.data_ptr() if sideband is not None else 0, int(value) & _WORD))
    device, stream = wrapper._device_and_stream(first)      # where the arrays live, the current device or not
    wrapper.library().sideaware_elementwise_batch(kernel_id, len(packed), b"".join(packed), device, stream)


def _rope_heads_many(tensors, freqs: torch.Tensor, backward: bool, positions: Optional[torch.Tensor] = None):
    first = tensors[0]
    assert first.dim() == 4, "activations are (B, T, heads, head_dim)"
    T, head_dim = first.shape[1], first.shape[3]
    if positions is not None:
        return _rope_many_at_positions(tensors, freqs, backward, positions, half=False)
    dtype = _ROPE_DTYPES.get(first.dtype)
    if dtype is None:
        raise TypeError("RoPE storage is float32, bfloat16 or float16")
    assert freqs.dtype == torch.float32 and tuple(freqs.shape) == (T, head_dim)
    for t in tensors:
        assert t.dim() == 4 and t.shape[1] == T and t.shape[3] == head_dim and t.dtype == first.dtype
    kid = _kernel("rope", (T, 0, 0, head_dim, dtype, "heads", backward), (("heads_at_launch", True),))
    elementwise_batch(kid, [(t.numel() * t.element_size(), [t], [t, freqs], None, t.shape[2]) for t in tensors])
    return tensors


def _rope_many_at_positions(tensors, freqs, backward: bool, positions: torch.Tensor, half: bool):
    first = tensors[0]
    B, T, head_dim = first.shape[0], first.shape[1], first.shape[3]
    dtype = _ROPE_DTYPES.get(first.dtype)
    if dtype is None:
        raise TypeError("RoPE storage is float32, bfloat16 or float16")
    assert freqs.dtype == torch.float32 and freqs.dim() == 2 and freqs.shape[1] == head_dim
    _check_positions(positions, B * T, first, freqs.shape[0])
    for t in tensors:
        assert t.dim() == 4 and t.is_contiguous() and t.shape[:2] == first.shape[:2] and t.shape[3] == head_dim \
            and t.dtype == first.dtype
    launch_time = (("heads_at_launch", True), ("positions", True))
    if half:
        kid = _kernel("rope_half", (1, 0, head_dim, dtype, backward), launch_time)
    else:
        kid = _kernel("rope", (1, 0, 0, head_dim, dtype, "heads", backward), launch_time)
    elementwise_batch(kid, [(t.numel() * t.element_size(), [t], [t, freqs], positions, t.shape[2]) for t in tensors])
    return tensors


def rope_forward_heads_many(tensors, freqs, positions=None):
    """Rotates several (B, T, heads, head_dim) tensors in place in ONE launch: q and k of a
    grouped-query model (different head counts, same T, head_dim and dtype) share a grid.
    ``positions`` as in :func:`rope_forward_heads`."""
    return _rope_heads_many(list(tensors), freqs, False, positions)


def rope_backward_heads_many(tensors, freqs, positions=None):
    return _rope_heads_many(list(tensors), freqs, True, positions)


def _rope_half(x: torch.Tensor, freqs: torch.Tensor, out: Optional[torch.Tensor], heads_first: bool,
               backward: bool, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    assert x.dim() == 4 and x.is_contiguous(), "activations are contiguous (B, T, heads, head_dim) or (B, heads, T, head_dim)"
    if heads_first:
        _, heads, T, head_dim = x.shape
    else:
        _, T, heads, head_dim = x.shape
    dtype = _ROPE_DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError("RoPE storage is float32, bfloat16 or float16")
    if positions is None:
        assert freqs.dtype == torch.float32 and tuple(freqs.shape) == (T, head_dim)
    else:
        assert not heads_first, "positions are per token of a (B, T, heads, head_dim) tensor"
        assert freqs.dtype == torch.float32 and freqs.dim() == 2 and freqs.shape[1] == head_dim
        _check_positions(positions, x.shape[0] * T, x, freqs.shape[0])
        T = 1                                   # the sequence length is not part of the compiled text
    if out is None:
        out = x
    assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()
    kid = _kernel("rope_half", (T, heads, head_dim, dtype, backward, heads_first), (("positions", positions is not None),))
    _elementwise(kid, out, None, None, None, x, freqs, None, None, positions, 0, 0, 0)
    return out


def rope_half_forward(x, freqs, out=None, heads_first: bool = False, positions=None):
    """RoPE for the half-split pair layout (element i of a head pairs with element
    i + head_dim/2, the "rotate_half" convention): (B, T, heads, head_dim), or
    (B, heads, T, head_dim) with ``heads_first``.  ``freqs`` is the same (T, head_dim) table the
    interleaved ops take ([t, 2i] = cos, [t, 2i+1] = sin of pair i).  In place unless ``out`` is given.
    ``positions`` as in :func:`rope_forward_heads`."""
    return _rope_half(x, freqs, out, heads_first, False, positions)


def rope_half_backward(dout, freqs, out=None, heads_first: bool = False, positions=None):
    return _rope_half(dout, freqs, out, heads_first, True, positions)


def rope_half_forward_many(tensors, freqs, backward: bool = False, positions=None):
    """Half-split RoPE of several (B, T, heads, head_dim) tensors in place in ONE launch (q and k
    of a grouped-query model).  ``positions`` as in :func:`rope_forward_heads`."""
    tensors = list(tensors)
    if positions is not None:
        return _rope_many_at_positions(tensors, freqs, backward, positions, half=True)
    first = tensors[0]
    T, head_dim = first.shape[1], first.shape[3]
    dtype = _ROPE_DTYPES.get(first.dtype)
    if dtype is None:
        raise TypeError("RoPE storage is float32, bfloat16 or float16")
    assert freqs.dtype == torch.float32 and tuple(freqs.shape) == (T, head_dim)
    for t in tensors:
        assert t.dim() == 4 and t.is_contiguous() and t.shape[1] == T and t.shape[3] == head_dim and t.dtype == first.dtype
    kid = _kernel("rope_half", (T, 0, head_dim, dtype, backward), (("heads_at_launch", True),))
    elementwise_batch(kid, [(t.numel() * t.element_size(), [t], [t, freqs], None, t.shape[2]) for t in tensors])
    return tensors


def freqs_cis_axes_table(sections, end: int, theta: float, order: str = "blocks") -> torch.Tensor:
    """(end, head_dim) fp32 table on the host, as :func:`freqs_cis_table` lays it out, for axes that
    each have a geometric series of frequencies of their own: the i-th pair of axis a turns by
    ``t * theta^(-i/sections[a])``.  (:func:`freqs_cis_table` itself is the table for axes that share one
    series over all pairs.)  Angles in 64 bits, rounded once."""
    axis = headers.rope_pair_axes(sections, order)
    seen = [0] * len(sections)
    freq = []
    for a in axis:
        freq.append(float(theta) ** (-seen[a] / sections[a]))
        seen[a] += 1
    angle = torch.arange(end, dtype=torch.float64)[:, None] * torch.tensor(freq, dtype=torch.float64)[None, :]
    return torch.stack([angle.cos(), angle.sin()], -1).reshape(end, 2 * len(axis)).float()


# What calls of the ops below need besides their pointers, by everything it depends on (shapes, types, devices and
# options, never a tensor): the checks of those are made once for each.
_PLANS_KEPT = 4096
_plans: Dict[Tuple, Tuple] = {}


def _keep_plan(key: Tuple, plan: Tuple) -> Tuple:
    if len(_plans) >= _PLANS_KEPT:
        _plans.clear()
    _plans[key] = plan
    return plan


# Workgroups finish in any order: an output may be an input itself, element for element, but no part of another array.
_OVERLAP = "an output overlaps another array of the call"


def _aligned(t: torch.Tensor, name: str) -> int:
    """Address of a tensor whose device is known: contiguous and 16-byte aligned."""
    assert t.is_contiguous(), name + " must be contiguous"
    ptr = t.data_ptr()
    assert not ptr & 15, name + " must be 16-byte aligned"
    return ptr


def _rope_axes_plan(shapes, out_shapes, dtypes, devices, freqs_shape, positions_shape, sections, half, order, backward):
    """The kernel, for each tensor its bytes and sideband value, and the bytes of the table and the positions."""
    first = shapes[0]
    assert len(first) == 4, "activations are (B, T, heads, head_dim)"
    B, T, _, head_dim = first
    dtype = _ROPE_DTYPES.get(dtypes[0])
    if dtype is None:
        raise TypeError("RoPE storage is float32, bfloat16 or float16")
    freqs_type, positions_type = dtypes[-2:]
    assert freqs_type == torch.float32 and len(freqs_shape) == 2 and freqs_shape[1] == head_dim, "the table is float32, (rows, head_dim)"
    if freqs_shape[0] * freqs_shape[1] * 4 >= 1 << 32:
        raise ValueError("the table of multi-axis RoPE is smaller than 4 GiB")
    assert positions_type == torch.int32, "positions are a contiguous int32 tensor"
    assert tuple(positions_shape) in ((B, T, len(sections)), (B * T, len(sections))), \
        "positions are (B, T, axes): one row of the table for each axis of every token"
    assert len(out_shapes) == len(shapes), "one output per tensor"
    for t, o in zip(shapes, out_shapes):
        assert len(t) == 4 and t[:2] == first[:2] and t[3] == head_dim, "tensors share B, T and head_dim"
        assert o == t, "an output is like its tensor"
    assert all(d == dtypes[0] for d in dtypes[:-2]), "tensors and outputs share one type"
    assert devices[0] >= 0 and all(d == devices[0] for d in devices), "tensors, outputs, table and positions live on one GPU"
    kid = _kernel("rope_axes", (head_dim, tuple(int(s) for s in sections), dtype, half, order, backward))
    size = 4 if dtype == "fp32" else 2
    sizes = [(t.numel() * size, headers.rope_axes_sideband(t[2], freqs_shape[0])) for t in shapes]
    return kid, sizes, freqs_shape[0] * freqs_shape[1] * 4, B * T * len(sections) * 4


def _rope_axes_many(tensors, freqs, positions, sections, half: bool, order: str, backward: bool, outs):
    tensors = list(tensors)
    outs = tensors if outs is None else list(outs)
    if torch.compiler.is_compiling():
        torch.ops.sideaware.rope_axes(tensors, freqs, positions, [int(s) for s in sections], bool(half), order, backward, outs)
    else:
        _rope_axes_launch(tensors, freqs, positions, sections, half, order, backward, outs)
    return outs


def _rope_axes_launch(tensors, freqs, positions, sections, half: bool, order: str, backward: bool, outs) -> None:
    every = tensors + outs + [freqs, positions]
    shapes, dtypes, devices = [t.shape for t in every], [t.dtype for t in every], [t.get_device() for t in every]
    n = len(tensors)
    assert positions.is_contiguous(), "positions are a contiguous int32 tensor"
    sections = tuple(sections)
    key = ("rope_axes", n, tuple(shapes), tuple(dtypes), tuple(devices), sections, bool(half), order, backward)
    plan = _plans.get(key)
    if plan is None:
        plan = _keep_plan(key, _rope_axes_plan(shapes[:n], shapes[n:-2], dtypes, devices, freqs.shape, positions.shape,
                                               sections, bool(half), order, backward))
    kid, sizes, table_bytes, where_bytes = plan
    if sizes[0][0]:                                            # all have elements, or none
        table, where = _aligned(freqs, "freqs"), positions.data_ptr()
        arrays = [(_aligned(o, "out"), _aligned(t, "x"), size) for t, o, (size, _) in zip(tensors, outs, sizes)]
        for i, (out, inp, size) in enumerate(arrays):
            end = out + size
            overlap = (out != inp and out < inp + size and inp < end or out < table + table_bytes and table < end
                       or out < where + where_bytes and where < end)
            for o, x, n_bytes in arrays[:i]:
                overlap = overlap or out < o + n_bytes and o < end or out < x + n_bytes and x < end or o < inp + size and inp < o + n_bytes
            if overlap:
                raise ValueError(_OVERLAP)
        packed = b"".join([_SEGMENT.pack(size, out, 0, 0, 0, inp, table, 0, 0, where, value & _WORD)
                           for (out, inp, size), (_, value) in zip(arrays, sizes)])
        device, stream = wrapper._device_and_stream(freqs)
        wrapper.library().sideaware_elementwise_batch(kid, n, packed, device, stream)


def rope_axes_forward_many(tensors, freqs, positions, sections, half: bool = False, order: str = "blocks", outs=None):
    """RoPE with a position of 1 to 3 axes (the time, height and width of an image's or video's patch) of
    several (B, T, heads, head_dim) tensors in ONE launch: q and k of a grouped-query model (different
    head counts, same B, T, head_dim and dtype).  In place unless ``outs`` is given; returns the outputs.  An
    output is its own tensor or shares no memory with any other, the table and the positions among them.

    ``freqs``: the (rows, head_dim) fp32 table of the ops with one position (``freqs_cis_table``, or
    ``freqs_cis_axes_table`` for axes with frequencies of their own), with a row for every position that
    occurs.  ``positions``: int32 (B, T, axes), contiguous; a position outside the table makes the pairs of
    its axis NaN.  ``sections``: how many of a head's head_dim/2 pairs each axis turns: in blocks of
    consecutive pairs (``order="blocks"``) or dealt to the axes in turn (``"turns"``).  ``half``: half-split
    pairs (element i with element i + head_dim/2), as :func:`rope_half_forward` has them, instead of
    neighbouring ones."""
    return _rope_axes_many(tensors, freqs, positions, sections, half, order, False, outs)


def rope_axes_backward_many(tensors, freqs, positions, sections, half: bool = False, order: str = "blocks", outs=None):
    """The gradients of :func:`rope_axes_forward_many` (``tensors`` are those of its outputs): the rotation
    by the opposite angles."""
    return _rope_axes_many(tensors, freqs, positions, sections, half, order, True, outs)


def rope_axes_forward(x, freqs, positions, sections, out=None, half: bool = False, order: str = "blocks"):
    """:func:`rope_axes_forward_many` of one tensor.  In place unless ``out`` is given."""
    return _rope_axes_many([x], freqs, positions, sections, half, order, False, None if out is None else [out])[0]


def rope_axes_backward(dout, freqs, positions, sections, out=None, half: bool = False, order: str = "blocks"):
    return _rope_axes_many([dout], freqs, positions, sections, half, order, True, None if out is None else [out])[0]


def dropout_threshold(p: float) -> int:
    """The probability to drop in units of 2^-16, rounded to nearest: what the dropout ops work with."""
    if not 0.0 <= p <= 1.0:
        raise ValueError("the probability to drop lies in [0, 1], got %r" % (p,))
    return int(math.floor(p * 65536.0 + 0.5))


def _dropout(x: torch.Tensor, p: float, seed: torch.Tensor, residual: Optional[torch.Tensor], out: Optional[torch.Tensor]):
    if torch.compiler.is_compiling():
        out = _like(out, x, "out")
        torch.ops.sideaware.dropout(x, p, seed, residual, out)
        return out
    return _dropout_launch(x, p, seed, residual, out)


def _dropout_launch(x: torch.Tensor, p: float, seed: torch.Tensor, residual: Optional[torch.Tensor], out: Optional[torch.Tensor]):
    threshold = dropout_threshold(p)
    dtype = _ROPE_DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError("dropout storage is float32, bfloat16 or float16")
    device = x.get_device()
    assert seed.dtype == torch.int64 and seed.numel() == 2 and seed.is_contiguous() and seed.get_device() == device, \
        "the seed is an int64 tensor of two values (seed, offset) on the activations' device"
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype and residual.get_device() == device, "the residual is like the activation"
    out = _like(out, x, "out")
    if x.numel():
        assert x.is_cuda, "x must be on the GPU"
        kid = _kernel("dropout", (dtype, residual is not None))
        size, to, first = x.numel() * x.element_size(), _aligned(out, "out"), _aligned(x, "x")
        second = 0 if residual is None else _aligned(residual, "residual")
        state = seed.data_ptr()
        if 0 < abs(to - first) < size or second and 0 < abs(to - second) < size or to < state + 16 and state < to + size:
            raise ValueError(_OVERLAP)
        device, stream = wrapper._device_and_stream(x)
        wrapper.library().sideaware_elementwise(kid, size, to, 0, 0, 0, first, second, 0, 0, state, threshold, 0, 0, device, stream)
    return out


def _dropout_node(x, p, seed, residual, out) -> None:
    _dropout_launch(x, p, seed, residual, out)


# Under torch.compile a call of these ops is one node of the graph, whose implementation is the eager call with all its
# checks (by then tensors have addresses): the same launch, and the same refusals.
_library = torch.library.Library("sideaware", "FRAGMENT")
_library.define("rope_axes(Tensor[] tensors, Tensor freqs, Tensor positions, int[] sections, bool half, str order, bool backward, Tensor(a!)[] outs) -> ()")
_library.define("dropout(Tensor x, float p, Tensor seed, Tensor? residual, Tensor(a!) out) -> ()")
_library.impl("rope_axes", _rope_axes_launch, "CUDA")
_library.impl("dropout", _dropout_node, "CUDA")


def dropout_forward(x, p: float, seed, residual=None, out=None):
    """``x / (1 - p)`` where an element is kept and 0 where it is dropped (with probability ``p``, rounded to
    a multiple of 2^-16), plus ``residual`` if one is given, rounded once to the tensors' type.  The mask
    is computed from the element's index and ``seed``, an int64 device tensor (seed, offset), and never
    stored: pass the same two to :func:`dropout_backward`.  A launch captured into a graph reads the
    tensor at every replay, so advancing the offset in place gives each replay a new mask.
    ``x`` may have any number of elements.  ``out`` may be ``x`` or ``residual``, but not overlap them otherwise, nor ``seed``."""
    return _dropout(x, p, seed, residual, out)


def dropout_backward(dout, p: float, seed, out=None):
    """The gradient of :func:`dropout_forward` with respect to ``x`` (that of the residual is ``dout``)."""
    return _dropout(dout, p, seed, None, out)


_GROUP_NORM_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {"none": 0, "silu": 1}


def _group_norm_plan(shape, dtype_of_x, device, params, groups: int, activation: str):
    """(batch, pixels, channels, type, weight_fp32, activation, bytes of workspace forward and backward) of a call, its
    sizes, types and devices checked; ``params`` are the (shape, type, device) of weight and bias, or None."""
    dtype = _GROUP_NORM_TYPES.get(dtype_of_x)
    if dtype is None:
        raise TypeError("group norm storage is float32, bfloat16 or float16")
    if activation not in _ACTIVATIONS:
        raise ValueError("the activation is 'none' or 'silu'")
    assert len(shape) >= 2, "activations are (N, ..., C), channels last"
    batch, channels = shape[0], shape[-1]
    if groups < 1 or channels < 1 or channels % groups:
        raise ValueError("%d groups do not divide %d channels" % (groups, channels))
    pixels = 1
    for n in shape[1:-1]:
        pixels *= n
    if pixels < 1:
        raise ValueError("a sample without pixels has no mean")
    params = [t for t in params if t is not None]
    for of_shape, of_type, of_device in params:
        assert of_type in (torch.float32, dtype_of_x) and of_type == params[0][1], "weight and bias are both float32 or both of the activations' type"
        assert tuple(of_shape) == (channels,) and of_device == device, "weight and bias have one value per channel, on the activations' device"
    weight_fp32 = 1 if not params or params[0][1] == torch.float32 else 0
    need = [0, 0]
    if batch and device >= 0:
        need = [wrapper.library().sideaware_group_norm_workspace(batch, pixels, channels, groups, dtype, backward, device) for backward in (0, 1)]
    return batch, pixels, channels, dtype, weight_fp32, _ACTIVATIONS[activation], need


def _group_norm_call(x: torch.Tensor, weight, bias, groups: int, activation: str):
    device = x.get_device()
    params = tuple(None if t is None else (t.shape, t.dtype, t.get_device()) for t in (weight, bias))
    key = ("group_norm", x.shape, x.dtype, device, params, groups, activation)
    plan = _plans.get(key)
    if plan is None:
        plan = _keep_plan(key, _group_norm_plan(x.shape, x.dtype, device, params, groups, activation))
    assert (weight is None or weight.is_contiguous()) and (bias is None or bias.is_contiguous()), "weight and bias are contiguous"
    return plan


def _may_allocate(what: str) -> None:
    """Under this library's allocator, memory that is allocated while a stream is being captured goes back to
    the pool when the tensor dies, while the graph still writes it."""
    if torch.compiler.is_compiling():                          # the tracer allocates
        return
    if wrapper._allocator_installed and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("under stream capture pass %s: the graph needs memory that outlives it" % what)


def _like(t, x: torch.Tensor, name: str) -> torch.Tensor:
    if t is None:
        _may_allocate(name)
        return torch.empty_like(x)
    assert t.shape == x.shape and t.dtype == x.dtype and t.get_device() == x.get_device(), name + " is like the activation"
    return t


def _workspace(workspace, need: int, x: torch.Tensor):
    """(address, bytes, tensor) of a call's workspace."""
    if workspace is None:
        if need == 0:
            return 0, 0, None
        _may_allocate("workspace")
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
        return workspace.data_ptr(), need, workspace
    assert workspace.get_device() == x.get_device(), "the workspace lives on the activations' device"
    return _aligned(workspace, "workspace"), workspace.numel() * workspace.element_size(), workspace


def group_norm_workspace(x: torch.Tensor, groups: int, backward: bool = False) -> int:
    """The bytes of ``workspace`` that :func:`group_norm_forward` (or backward) of ``x`` needs; may be 0."""
    return _group_norm_call(x, None, None, groups, "none")[6][1 if backward else 0]


def _group_norm_failed(what: str):
    raise RuntimeError("%s: %s" % (what, wrapper.sideaware_last_error()))


def _check_stats(stats: torch.Tensor, batch: int, groups: int, x: torch.Tensor) -> None:
    assert stats.shape == (batch, groups, 2) and stats.dtype == torch.float32 and stats.is_contiguous() and stats.get_device() == x.get_device(), \
        "stats are float32 (N, groups, 2)"


def group_norm_forward(x, weight, bias, groups: int, eps: float = 1e-5, activation: str = "none", out=None, stats=None, workspace=None):
    """Group norm over (N, ..., C) activations, channels last: ``act((x - mean) / sqrt(var + eps) * weight + bias)``
    with mean and variance over a sample's pixels and the C / groups channels of a group, and ``act`` either
    "none" or "silu".  ``weight`` and ``bias`` are (C,), both float32 or both of x's type, or None.
    Returns (y, stats), stats being float32 (N, groups, 2): mean and 1 / sqrt(var + eps), which
    :func:`group_norm_backward` takes.  (A channels-last (N, C, H, W) tensor is ``t.permute(0, 2, 3, 1)``.)

    ``out`` (may be ``x``), ``stats`` and ``workspace`` (:func:`group_norm_workspace` bytes, of any type) are
    allocated unless given.  Under stream capture with this library's allocator they have to be given, and calls that can
    overlap, such as two graphs' replays, each need their own."""
    batch, pixels, channels, dtype, weight_fp32, act, need = _group_norm_call(x, weight, bias, groups, activation)
    out = _like(out, x, "out")
    if stats is None:
        _may_allocate("stats")
        stats = torch.empty((batch, groups, 2), dtype=torch.float32, device=x.device)
    else:
        _check_stats(stats, batch, groups, x)
    if batch == 0:
        return out, stats
    assert x.is_cuda, "x must be on the GPU"
    ws_ptr, ws_bytes, keep = _workspace(workspace, need[0], x)
    device, stream = wrapper._device_and_stream(x)
    if wrapper.library().sideaware_group_norm_forward(
            _aligned(out, "out"), stats.data_ptr(), _aligned(x, "x"), weight.data_ptr() if weight is not None else None,
            bias.data_ptr() if bias is not None else None, batch, pixels, channels, groups, eps, act, dtype, weight_fp32, ws_ptr, ws_bytes, device, stream):
        _group_norm_failed("group_norm_forward")
    return out, stats


def group_norm_backward(dout, x, weight, bias, stats, groups: int, activation: str = "none", out=None, dweight=None, dbias=None, workspace=None):
    """The gradients of :func:`group_norm_forward`: (dx, dweight, dbias), the latter two of weight's type and summed
    over samples and pixels (None where weight or bias is None).  ``stats`` is what the forward call returned.
    ``out`` may be ``dout``.  ``out``, ``dweight``, ``dbias`` and ``workspace`` are allocated unless given, as for the
    forward call."""
    batch, pixels, channels, dtype, weight_fp32, act, need = _group_norm_call(x, weight, bias, groups, activation)
    assert dout.shape == x.shape and dout.dtype == x.dtype and dout.get_device() == x.get_device(), "the gradient is like the activation"
    _check_stats(stats, batch, groups, x)
    out = _like(out, x, "out")
    assert dweight is None or weight is not None, "dweight goes with a weight"
    assert dbias is None or bias is not None, "dbias goes with a bias"
    dweight = None if weight is None else _like(dweight, weight, "dweight")
    dbias = None if bias is None else _like(dbias, bias, "dbias")
    assert (dweight is None or dweight.is_contiguous()) and (dbias is None or dbias.is_contiguous()), "dweight and dbias are contiguous"
    if batch == 0:
        for t in (dweight, dbias):
            if t is not None:
                t.zero_()
        return out, dweight, dbias
    assert x.is_cuda, "x must be on the GPU"
    ws_ptr, ws_bytes, keep = _workspace(workspace, need[1], x)
    device, stream = wrapper._device_and_stream(x)
    if wrapper.library().sideaware_group_norm_backward(
            _aligned(out, "out"), dweight.data_ptr() if dweight is not None else None, dbias.data_ptr() if dbias is not None else None,
            _aligned(dout, "dout"), _aligned(x, "x"), weight.data_ptr() if weight is not None else None,
            bias.data_ptr() if bias is not None else None, stats.data_ptr(),
            batch, pixels, channels, groups, act, dtype, weight_fp32, ws_ptr, ws_bytes, device, stream):
        _group_norm_failed("group_norm_backward")
    return out, dweight, dbias


def scale_bias_bf16(x: torch.Tensor, scale_bias: torch.Tensor, out: Optional[torch.Tensor] = None):
    """bf16 ``y = x*scale + bias`` in fp32, rounded to nearest even.  ``scale_bias`` is a device
    tensor of two fp32 values, read by the kernel, so changing them costs no compile."""
    assert x.dtype == torch.bfloat16 and scale_bias.dtype == torch.float32 and scale_bias.numel() >= 2
    if out is None:
        out = torch.empty_like(x)
    kid = _kernel("scale_bias_bf16")
    _elementwise(kid, out, None, None, None, x, None, None, None, scale_bias, 0, 0, 0)
    return out


def mxfp8_quantize(x: torch.Tensor, q: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None):
    """bf16 -> MXFP8: returns (E4M3 bytes as a uint8 tensor shaped like x, E8M0 scale bytes, one
    per 32 consecutive elements).  ``x.numel()`` must be a multiple of 32."""
    assert x.dtype == torch.bfloat16 and x.is_contiguous() and x.numel() % 32 == 0
    if q is None:
        q = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    if scales is None:
        scales = torch.empty(x.numel() // 32, dtype=torch.uint8, device=x.device)
    assert q.dtype == torch.uint8 and q.numel() == x.numel() and scales.numel() == x.numel() // 32
    kid = _kernel("mxfp8_quantize")
    device, stream = wrapper._device_and_stream()
    # num_bytes is the byte length of the wider array, the bf16 input, which the custom-op wrapper
    # cannot know (it sizes the launch from out0, as the reference's does): call the C entry point.
    # the sideband value is the number of 16-byte vectors: the op gathers a wave's 16 scale bytes
    # into one store wherever the whole wave lies inside the array
    wrapper.library().sideaware_elementwise(kid, x.numel() * 2, q.data_ptr(), 0, 0, 0, x.data_ptr(), 0, 0, 0,
                                            scales.data_ptr(), min(x.numel() // 8, 2 ** 31 - 1), 0, 0, device, stream)
    return q, scales


def mxfp8_dequantize(q: torch.Tensor, scales: torch.Tensor, out: Optional[torch.Tensor] = None):
    """MXFP8 -> bf16: ``q`` E4M3 bytes (uint8), ``scales`` one E8M0 byte per 32 elements."""
    assert q.dtype == torch.uint8 and scales.dtype == torch.uint8 and q.is_contiguous() and scales.is_contiguous()
    assert q.numel() % 32 == 0 and scales.numel() == q.numel() // 32
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    assert out.dtype == torch.bfloat16 and out.numel() == q.numel()
    kid = _kernel("mxfp8_dequantize")
    # out0 is the wider array, so the custom op's own sizing (from out0) is the right one
    _elementwise(kid, out, None, None, None, q, None, None, None, scales, 0, 0, 0)
    return out


def fill_int32(out: torch.Tensor, value: int):
    """Writes a 32-bit pattern over ``out`` (byte size a multiple of 16): an output-only op."""
    kid = _kernel("fill")
    _elementwise(kid, out, None, None, None, None, None, None, None, None, int(value), 0, 0)
    return out
