"""Operators of packed token sequences: rotary positions and causal attention.

A packed batch lays sequences of different lengths out back to back, ``[tokens, heads, dim]``
without a padded row; ``offsets`` (int32 on the tensors' device, ``sequences + 1`` entries, the
first one 0) says where each begins.

``rotary_embed`` turns queries and keys by their positions: whole or fractional, one per token or
one per axis, both pair layouts, all of a head or its leading part, with frequencies that
``rotary_frequencies`` may scale for contexts beyond the trained ones.  ``packed_attention`` is
causal softmax attention with grouped key heads; the queries of a sequence are the last rows of
its keys, so one call covers a whole prompt, a prompt that goes on behind a cached part, and a
single token against a cache with room behind every sequence.

Both run in CUDA kernels on a B200 (``csrc/rotary.cu``, ``csrc/packed_attention*.cu``), forward and
gradient, and never synchronise with the device; elsewhere, and for types and head sizes that the
kernels do not cover, they evaluate the PyTorch definitions of :mod:`agentgarten_b200.ops.reference`
(whose packed attention reads the offsets on the host).
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import native, reference

__all__ = ["RotaryFrequencies", "packed_attention", "rotary_embed", "rotary_frequencies"]

SCALINGS = ("linear", "ntk", "yarn")
_KERNEL_TYPES = (torch.bfloat16, torch.float16, torch.float32)


# ------------------------------------------------------------------------------- rotary positions
@dataclass(frozen=True)
class RotaryFrequencies:
    """What ``rotary_embed`` turns by: ``turns`` FP64 ``[slots]``, turns (of 2 pi) per position;
    ``amplitude`` that multiplies the turned values; ``axis`` int32 ``[slots]``, which column of
    the positions turns each slot (``None``: positions have one value per token)."""

    turns: torch.Tensor
    amplitude: float = 1.0
    axis: torch.Tensor | None = None

    @property
    def rotary_dim(self) -> int:
        return 2 * self.turns.shape[0]


def rotary_frequencies(rotary_dim: int, theta: float = 10_000.0, *, scaling: str | None = None,
                       factor: float = 1.0, trained_positions: int | None = None,
                       fast_turns: float = 32.0, slow_turns: float = 1.0,
                       sections: tuple[int, int, int] | None = None,
                       device: torch.device | str | None = None) -> RotaryFrequencies:
    """Frequencies ``theta ** (-2 j / rotary_dim)`` for the first ``rotary_dim`` elements of a head.

    ``scaling`` stretches them for contexts ``factor`` times the trained one: ``"linear"`` divides
    the positions; ``"ntk"`` raises theta so that the slowest slot is divided by ``factor`` and the
    fastest stays; ``"yarn"`` (Peng et al. 2023) keeps the slots that make more than ``fast_turns``
    turns over ``trained_positions``, divides those below ``slow_turns``, blends between, and
    multiplies the turned values by ``0.1 ln(factor) + 1``.

    ``sections`` (time, row, column) makes the slots of three position axes, interleaved as the
    towers' tables have them: slot ``j`` belongs to axis ``j % 3`` while ``j < 3 * sections[axis]``,
    else to time.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling is not None and scaling not in SCALINGS:
        raise ValueError(f"unknown rotary scaling {scaling!r}: one of {', '.join(SCALINGS)}")
    if not theta > 1 or not factor >= 1 or not math.isfinite(theta * factor):
        raise ValueError("theta must be above 1 and the scaling factor at least 1")
    slots = rotary_dim // 2
    slot = torch.arange(slots, dtype=torch.float64)
    base, amplitude = float(theta), 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs at least two slots")
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    inverse = base ** (-slot / slots)
    if scaling == "linear":
        inverse = inverse / factor
    elif scaling == "yarn":
        if not trained_positions or not fast_turns > slow_turns > 0:
            raise ValueError("yarn scaling needs trained_positions and fast_turns > slow_turns > 0")

        def slot_of(turns: float) -> float:  # the slot that makes this many turns over the trained range
            return slots * math.log(trained_positions / (turns * 2 * math.pi)) / math.log(theta)

        low = max(0, math.floor(slot_of(fast_turns)))
        high = min(rotary_dim - 1, math.ceil(slot_of(slow_turns)))
        kept = 1 - ((slot - low) / max(high - low, 1e-3)).clamp(0, 1)
        inverse = inverse * kept + inverse / factor * (1 - kept)
        amplitude = 0.1 * math.log(factor) + 1.0
    axis = None
    if sections is not None:
        if len(sections) != 3 or any(s < 0 for s in sections):
            raise ValueError("sections are three counts: time, row, column")
        index = torch.arange(slots)
        axis = torch.zeros(slots, dtype=torch.int32)
        for which in (1, 2):
            axis[(index % 3 == which) & (index < 3 * sections[which])] = which
        axis = axis.to(device)
    return RotaryFrequencies((inverse / (2 * math.pi)).to(device), amplitude, axis)


def rotary_embed(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor,
                 frequencies: RotaryFrequencies, *, interleaved: bool = False):
    """Query and key turned by their positions, in one pass: ``(query, key)`` as new tensors.

    ``query`` ``[..., heads, dim]`` and ``key`` ``[..., kv_heads, dim]`` (or ``None``) are bf16,
    fp16 or fp32 and share the leading dimensions; ``positions`` (int32, int64 or fp32) has these
    leading dimensions, and a last one of three axes where the frequencies have axes.  The first
    ``frequencies.rotary_dim`` elements of a head are turned, the others copied; a pair is
    ``(x[j], x[j + rotary_dim / 2])``, or ``(x[2 j], x[2 j + 1])`` with ``interleaved``.  Angles
    are exact for any position that the type of ``positions`` holds; the turn is 32-bit arithmetic,
    rounded once.  Differentiable in query and key.
    """
    f = frequencies
    if query.is_cuda and native.use(query, dtypes=_KERNEL_TYPES):
        out = native.ext().rotary_embed(query, key, positions, f.turns, f.axis, f.amplitude, interleaved)
        if out is not None:
            return out[0], (out[1] if key is not None else None)
    given = [query] if key is None else [query, key]
    lead = query.shape[:-2]
    for name, t in zip(("query", "key"), given):
        if t.dim() < 3 or t.shape[:-2] != lead or t.shape[-1] != query.shape[-1] or t.shape[-2] == 0:
            raise ValueError(f"rotary_embed: {name} {tuple(t.shape)} is not [..., heads, dim] over {tuple(lead)}")
        if t.dtype != query.dtype or t.dtype not in (*_KERNEL_TYPES, torch.float64):
            raise TypeError(f"rotary_embed: {name} is {t.dtype}: both are bf16, fp16, fp32 or fp64")
    if f.rotary_dim > query.shape[-1]:
        raise ValueError(f"rotary_embed: {f.rotary_dim} elements to turn in heads of {query.shape[-1]}")
    want = tuple(lead) if f.axis is None else (*lead, 3)
    if tuple(positions.shape) != want:
        raise ValueError(f"rotary_embed: positions {tuple(positions.shape)} are not {want}")
    if positions.dtype not in (torch.int32, torch.int64, torch.float32):
        raise TypeError(f"rotary_embed: positions are int32, int64 or fp32, not {positions.dtype}")
    if any(t.device != query.device for t in (*given, positions, f.turns)):
        raise ValueError("rotary_embed: query, key, positions and frequencies are on one device")
    turned = [reference.rotary_embed(t, positions, f.turns, f.amplitude, f.axis, interleaved) for t in given]
    return turned[0], (turned[1] if key is not None else None)


# ---------------------------------------------------------------------------- packed attention
def packed_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, q_offsets: torch.Tensor,
                     k_offsets: torch.Tensor | None = None, *, k_lengths: torch.Tensor | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """Causal softmax attention over packed sequences: ``[total_q, heads, dim]``.

    ``query`` ``[total_q, heads, dim]``; ``key`` and ``value`` ``[total_k, kv_heads, dim]`` with
    ``heads`` a multiple of ``kv_heads``.  Sequence ``s`` owns the query rows ``q_offsets[s] :
    q_offsets[s + 1]`` and the first ``k_lengths[s]`` (default: all) of the key rows ``k_offsets[s]
    : k_offsets[s + 1]`` (default: its query rows).  Its queries are the *last* rows of its keys:
    query ``i`` of ``n`` sees the keys up to ``keys - n + i``.  A query that sees no key gives zeros,
    and so do rows behind the last sequence.  What lies in key rows that belong to no sequence, to
    another one or behind ``k_lengths`` has no influence, whatever it holds.  A NaN or an infinity
    among a sequence's own rows may spread within that sequence: a value to queries that stop short
    of it within the same 128 keys, and in the gradient a query to keys behind it within the same
    tile of queries.

    The offsets stay on the device.  The kernels check them; a sequence whose offsets do not fit is
    skipped and reported through the kernel status word.  ``scale`` defaults to ``dim ** -0.5``.
    Differentiable in query, key and value.  Scores, statistics and sums are FP32; probabilities
    are rounded to the tensors' type where they enter a matrix product.
    """
    if query.is_cuda and native.use(query, dtypes=_KERNEL_TYPES[:2]):
        out = native.ext().packed_attention(query, key, value, q_offsets, k_offsets, k_lengths, scale)
        if out is not None:
            return out
    if query.dim() != 3 or key.dim() != 3 or value.shape != key.shape or query.shape[-1] != key.shape[-1]:
        raise ValueError(f"packed_attention: query {tuple(query.shape)}, key {tuple(key.shape)} and value "
                         f"{tuple(value.shape)} are not [total, heads, dim] with one dim")
    heads, dim = query.shape[1], query.shape[2]
    if key.shape[1] == 0 or heads == 0 or heads % key.shape[1] or dim == 0:
        raise ValueError(f"packed_attention: {heads} query heads are not a multiple of {key.shape[1]} key heads")
    if query.dtype != key.dtype or query.dtype != value.dtype or not query.dtype.is_floating_point:
        raise TypeError("packed_attention: query, key and value have one floating type")
    if k_offsets is None:
        if query.shape[0] != key.shape[0]:
            raise ValueError("packed_attention: k_offsets are needed where keys and queries are not the same rows")
        k_offsets = q_offsets
    lists = [q_offsets, k_offsets] if k_lengths is None else [q_offsets, k_offsets, k_lengths]
    for t in lists:
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise TypeError("packed_attention: offsets and lengths are contiguous int32 vectors")
    if q_offsets.shape[0] < 1 or k_offsets.shape != q_offsets.shape or (
            k_lengths is not None and k_lengths.shape[0] != q_offsets.shape[0] - 1):
        raise ValueError("packed_attention: sequences + 1 offsets of queries and of keys, and one length a sequence")
    if any(t.device != query.device for t in (key, value, *lists)):
        raise ValueError("packed_attention: all tensors are on one device")
    if max(query.shape[0], key.shape[0]) >= 2 ** 31 - 256:
        raise ValueError("packed_attention: rows are counted in 32 bits")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError("packed_attention: scale is positive")
    return reference.packed_attention(query, key, value, q_offsets, k_offsets, k_lengths, scale)
