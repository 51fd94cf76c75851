"""rotary_embedding, rotary_embedding_axes: rotary positions on queries and keys, on one axis or
several, and their gradient.

What produces the ``query_rope`` / ``key_rope`` arguments of the attention operators
(interleaved pairs, 64 wide) and the rotated part of the index queries and keys (half layout,
part of the head).  No counterpart in the reference, which takes rotated tensors.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _host as H
from ._lib import (BIND_AXES, BIND_ROTARY, DSA_DTYPE_FP32, ROTARY_MAX_AXES, RotaryAxesParams, RotaryParams, binding,
                   check, lib, ptr, remember, report_ptr, stream_ptr)

_MAX_DIM = 256
LAYOUTS = ("interleaved", "half")
ORDERS = ("blocks", "cycled")


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original_positions=4096,
                       beta_fast=32.0, beta_slow=1.0):
    """Angle per position of each of the dim / 2 pairs, base^(-2 i / dim), scaled for contexts
    longer than trained on: ``"linear"`` divides every angle by ``factor``; ``"ntk"`` raises the
    base by factor^(dim / (dim - 2)); ``"yarn"`` keeps the pairs that turn more than
    ``beta_fast`` times within ``original_positions``, divides those that turn less than
    ``beta_slow`` times, and blends between."""
    if dim < 2 or dim % 2 or dim > _MAX_DIM:
        raise ValueError(f"dim must be even, 2..{_MAX_DIM}, got {dim}")
    if not base > 1.0:
        raise ValueError(f"base must be above 1, got {base}")
    if not factor > 0.0:
        raise ValueError(f"factor must be positive, got {factor}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unsupported scaling {scaling!r}")
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs a dim above 2")
        base = base * factor ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        return [f / factor for f in freq]
    if scaling != "yarn":
        return freq
    if original_positions < 1 or beta_slow <= 0.0 or beta_fast < beta_slow:
        raise ValueError("yarn needs original_positions >= 1 and beta_fast >= beta_slow > 0")

    def pair_of(turns):
        return dim * math.log(original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low = max(0, math.floor(pair_of(beta_fast)))
    high = min(dim - 1, math.ceil(pair_of(beta_slow)))
    span = max(high - low, 0.001)
    ramp = [min(1.0, max(0.0, (i - low) / span)) for i in range(dim // 2)]
    return [f / factor * r + f * (1.0 - r) for f, r in zip(freq, ramp)]


def rotary_table(max_positions, dim, base=10000.0, scaling=None, factor=1.0, original_positions=4096,
                 beta_fast=32.0, beta_slow=1.0, amplitude=1.0, device=None) -> torch.Tensor:
    """fp32 table [max_positions, dim]: row p holds amplitude * cos(p f_i), then amplitude *
    sin(p f_i), with the frequencies of :func:`rotary_frequencies`; angles are formed in 64 bits.
    Made once and kept beside the weights."""
    if max_positions < 1:
        raise ValueError(f"max_positions must be positive, got {max_positions}")
    freq = rotary_frequencies(dim, base, scaling, factor, original_positions, beta_fast, beta_slow)
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise ValueError("all tensors must be CUDA tensors (no CPU fallback)")
    with torch.cuda.device(dev):
        table = torch.empty((int(max_positions), dim), dtype=torch.float32, device=dev)
        check(lib().dsa_rotary_table(ptr(table), int(max_positions), dim, (ctypes.c_double * len(freq))(*freq),
                                     float(amplitude), stream_ptr(table.device)), "dsa_rotary_table")
    return table


def _token_strides(t: torch.Tensor):
    """(batch, token, head) strides of a [B, S, N, H] or [T, N, H] tensor."""
    return (0, *t.stride()[:2]) if t.dim() == 3 else tuple(t.stride()[:3])


def _plan(x, table, positions, layout, offset, inverse, out, axes=None):
    """Check the arguments and fill in what their shapes decide; `axes`: how many axes the positions
    have, in a dim of their own."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if x.dim() not in (3, 4):
        raise ValueError("x must be [B, S, N, H] or [T, N, H]")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"unsupported dtype {x.dtype}: expected bfloat16, float16 or float32")
    if table.dim() != 2 or table.dtype != torch.float32:
        raise ValueError("table must be a float32 [max_positions, dim] tensor (rotary_table)")
    dim = table.shape[1]
    if dim < 2 or dim % 2 or dim > _MAX_DIM or table.shape[0] < 1:
        raise ValueError(f"the table's dim must be even, 2..{_MAX_DIM}, got {dim}")
    if offset < 0 or offset + dim > x.shape[-1]:
        raise ValueError(f"offset {offset} + dim {dim} exceed the head's {x.shape[-1]} values")
    shape = (*(() if axes is None else (axes,)), *x.shape[:-2])
    if tuple(positions.shape) != shape:
        raise ValueError(f"positions must be {shape}, got {tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    H.require_cuda(x, table, positions, out)
    if table.device != x.device or positions.device != x.device:
        raise ValueError("all tensors must be on one device")
    if out is not None:
        if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or out.stride(-1) != 1:
            raise ValueError("out must have x's shape, dtype and device, and a contiguous last dim")
        if H.self_overlap(out):
            raise ValueError("out must not be an expanded tensor")
    p = RotaryParams()
    p.batch, p.s = (1, x.shape[0]) if x.dim() == 3 else x.shape[:2]
    p.heads, p.head_dim, p.offset, p.dim = x.shape[-2], x.shape[-1], int(offset), dim
    p.max_positions = table.shape[0]
    p.x_batch_stride, p.x_token_stride, p.x_head_stride = _token_strides(x)
    o = torch.empty(x.shape, dtype=x.dtype, device="meta") if out is None else out
    p.out_batch_stride, p.out_token_stride, p.out_head_stride = _token_strides(o)
    p.half_layout, p.inverse = int(layout == "half"), int(bool(inverse))
    p.dtype = DSA_DTYPE_FP32 if x.dtype == torch.float32 else H.dtype_code(x)
    return bytes(p)


def _fill(p, x, table, positions, out):
    """Put the addresses in: (out, whether x, table and positions went in as they were given, what has to
    live until the launch)."""
    given = (x, table, positions)
    if x.stride(-1) != 1:
        if out is x:
            raise ValueError("a rotation in place needs a contiguous last dim")
        x = x.contiguous()
        p.x_batch_stride, p.x_token_stride, p.x_head_stride = _token_strides(x)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out is not x and H.overlap(out, x):
        raise ValueError("out overlaps x (pass x itself to rotate in place)")
    if positions.dtype != torch.int32:   # a position past 32 bits stays outside the table
        positions = positions.clamp(-1, 0x7fffffff).to(torch.int32)
    positions = positions.contiguous()
    table = table.contiguous()
    p.x, p.out = x.data_ptr(), out.data_ptr()
    p.positions, p.table = positions.data_ptr(), table.data_ptr()
    return out, all(a is b for a, b in zip(given, (x, table, positions))), (x, table, positions)


def rotary_embedding(x, table, positions, layout="interleaved", offset=0, inverse=False, out=None):
    """Rotate ``x`` [B, S, N, H] (``positions`` [B, S]) or [T, N, H] (``positions`` [T]): of each
    head the values ``offset`` .. ``offset + table.shape[1]`` turn by the angles of the token's
    position, the others are copied.  ``layout`` "interleaved" pairs (2 i, 2 i + 1), "half"
    pairs (i, i + dim / 2).  ``inverse`` turns back by the same table, amplitude kept: the
    gradient with respect to ``x`` of a rotation is the inverse rotation of the gradient.

    bf16, fp16 or fp32; any strides with a contiguous last dim.  ``out`` (same shape and type;
    ``x`` itself for a rotation in place) receives the result, else a new tensor.  A position
    outside the table gives a zero row and is reported by ``check_device_errors``.
    """
    args = (x, table, positions, layout, offset, bool(inverse), out)
    fast = binding()
    if fast is not None:
        done = fast.rotary(*args)
        if done is not None:
            return done
    template = _plan(x, table, positions, layout, offset, inverse, out)
    index = x.get_device()
    if H.current_device() != index:
        with torch.cuda.device(index):
            return rotary_embedding(x, table, positions, layout, offset, inverse, out)
    p = RotaryParams.from_buffer_copy(template)
    out, as_given, keep = _fill(p, x, table, positions, out)
    p.error_flag = report_ptr(index)
    check(lib().dsa_rotary(p, H.raw_stream(index)), "dsa_rotary")
    if as_given:
        remember(BIND_ROTARY, index, *args, template, b"", 0)
    return out


def rotary_axes(sections, order="blocks"):
    """The axis of each of the sum(sections) pairs, of which ``sections[a]`` turn by axis a.  "blocks":
    the first ``sections[0]`` pairs by axis 0, the next by axis 1, and so on.  "cycled": pair i by axis
    i % len(sections) as long as that axis has pairs left, by axis 0 from then on, so that each axis
    has fast and slow pairs; it needs ``sections[a]`` turns of every axis but the first."""
    try:
        sections = tuple(int(n) for n in sections)
    except TypeError:
        raise ValueError(f"sections must be a sequence of numbers, got {sections!r}") from None
    axes, half = len(sections), sum(sections)
    if not 1 <= axes <= ROTARY_MAX_AXES or min(sections) < 1:
        raise ValueError(f"sections must be 1..{ROTARY_MAX_AXES} positive numbers, got {sections}")
    if order not in ORDERS:
        raise ValueError(f"order must be one of {ORDERS}, got {order!r}")
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    if any(axes * (n - 1) + a >= half for a, n in enumerate(sections) if a):
        raise ValueError(f"sections {sections} cannot take turns: an axis has more pairs than turns")
    return [i % axes if i < axes * sections[i % axes] else 0 for i in range(half)]


def _axes_plan(x, table, positions, sections, layout, order, offset, inverse, out):
    axis_of = rotary_axes(sections, order)
    if table.dim() == 2 and 2 * len(axis_of) != table.shape[1]:
        raise ValueError(f"sections {tuple(sections)} must add up to the table's {table.shape[1] // 2} pairs")
    p = RotaryAxesParams()
    p.rotary = RotaryParams.from_buffer_copy(_plan(x, table, positions, layout, offset, inverse, out, len(sections)))
    p.axes = len(sections)
    for i, a in enumerate(axis_of):
        p.axis_of[i] = a
    return bytes(p)


def rotary_embedding_axes(x, table, positions, sections, layout="interleaved", order="blocks", offset=0,
                          inverse=False, out=None):
    """:func:`rotary_embedding` with positions on several axes (time, height and width of pictures and
    films): ``positions`` is [A, B, S] for ``x`` [B, S, N, H] or [A, T] for [T, N, H], A up to 4, and of
    the pairs of each head ``sections[a]`` turn by axis a's position, pair i by column i of the table
    as there.  ``order`` says which, see :func:`rotary_axes`; ``sections`` add up to
    ``table.shape[1] / 2``.  Text has the same position on every axis, and gives what
    ``rotary_embedding`` gives.

    A position outside the table on any axis gives a zero row and is reported by
    ``check_device_errors``.
    """
    sections = tuple(sections) if isinstance(sections, (list, tuple)) else sections
    args = (x, table, positions, sections, layout, order, offset, bool(inverse), out)
    fast = binding()
    if fast is not None:
        done = fast.axes(*args)
        if done is not None:
            return done
    template = _axes_plan(*args)
    index = x.get_device()
    if H.current_device() != index:
        with torch.cuda.device(index):
            return rotary_embedding_axes(x, table, positions, sections, layout, order, offset, inverse, out)
    p = RotaryAxesParams.from_buffer_copy(template)
    out, as_given, keep = _fill(p.rotary, x, table, positions, out)
    p.rotary.error_flag = report_ptr(index)
    check(lib().dsa_rotary_axes(p, H.raw_stream(index)), "dsa_rotary_axes")
    if as_given:
        remember(BIND_AXES, index, *args, template, b"", 0)
    return out
