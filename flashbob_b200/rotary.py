"""Rotary positions for the heads that `sdpa_bob` and the paged cache take.

    rotary = Rotary(head_dim=128, theta=10000.0)
    q, k = apply_rotary(q, k, rotary)                      # training: positions 0 ... N - 1
    out = sdpa_bob(q, k, v, is_causal=True)

A pair of elements at position t is turned by t * frequency; the gradient turns back, so the operation can be
differentiated any number of times, as second-order steps need.  The same `Rotary` goes to `append_kv` and `sdpa_paged`
(flashbob_b200/paged.py), which turn keys and queries on their way.

CUDA tensors go through libbob_sm100.so (csrc/rotary.cuh); CPU tensors take plain tensor operations, angles in 64 bits.  On the
GPU a frequency is kept as a 64-bit fraction of a turn, and position * fraction is taken modulo a turn in integers: off by
2^-64 of a turn per position, 8e-10 radians at position 2^31 and 4e-7 at 2^40.  16-bit results take the angle and its sines in
fp32, off by 8e-7 together; keys for a 4-bit cache are turned in 64 bits.
"""

from __future__ import annotations

import ctypes
import math
import numbers
from fractions import Fraction

import torch

from . import _lib, _native, ops
from .interface import _CPU_DTYPES, _CUDA_DTYPES, _CUDA_HEAD_DIMS, _as_count

__all__ = ["Rotary", "apply_rotary"]

_MAX_PAIRS = 64
# 2^256 / (2 pi), for turns as whole numbers of 2^-64
_TURN = round(2 ** 255 / Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803"))
_SCALINGS = (None, "linear", "ntk", "yarn")


def _number(name, value, *, low=0.0):
    if isinstance(value, bool) or not isinstance(value, numbers.Real):
        raise TypeError(f"{name} must be a number, got {value!r}")
    if not math.isfinite(value) or value <= low:
        raise ValueError(f"{name} must be finite and greater than {low:g}, got {value!r}")
    return float(value)


class Rotary:
    """Frequencies of a rotary position embedding; a plain value that can be shared between layers, devices and streams.

    The first `rotary_dim` elements of a head turn (default: all), in pairs (i, i + rotary_dim / 2) or, `interleaved`,
    (2 i, 2 i + 1); the others stay.  Pair i turns by theta ** (-2 i / rotary_dim) per position.  For contexts longer than
    a model was trained on, `scaling` with `factor` changes the frequencies:

      "linear"  all divided by factor
      "ntk"     theta multiplied by factor ** (rotary_dim / (rotary_dim - 2)): the slowest pair is divided by factor, the
                fastest stays
      "yarn"    divided by factor where a pair turns less than beta_slow times in `original_length` positions, unchanged
                where it turns more than beta_fast times, a blend between; the result is multiplied by
                `attention_factor` (default 0.1 ln factor + 1)

    `frequencies` gives them one by one instead (radians per position, rotary_dim / 2 numbers).
    """

    __slots__ = ("head_dim", "rotary_dim", "interleaved", "frequencies", "attention_factor", "_packed")

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, theta: float = 10000.0, interleaved: bool = False,
                 scaling: str | None = None, factor: float = 1.0, original_length: int | None = None, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attention_factor: float | None = None, frequencies=None):
        self.head_dim = _as_count("head_dim", head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else _as_count("rotary_dim", rotary_dim)
        if not 0 < self.rotary_dim <= min(self.head_dim, 2 * _MAX_PAIRS) or self.rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even, positive and at most head_dim={self.head_dim} and {2 * _MAX_PAIRS}, got {self.rotary_dim}")
        if not isinstance(interleaved, bool):
            raise TypeError(f"interleaved must be bool, got {type(interleaved).__name__}")
        self.interleaved = interleaved
        if scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {_SCALINGS}, got {scaling!r}")
        theta, factor = _number("theta", theta), _number("factor", factor)
        gain = 1.0
        if frequencies is not None:
            if scaling is not None:
                raise ValueError("frequencies are given: scaling has nothing to change")
            freqs = [float(f) for f in frequencies]
            if len(freqs) != self.rotary_dim // 2 or not all(math.isfinite(f) for f in freqs):
                raise ValueError(f"frequencies must be {self.rotary_dim // 2} finite numbers")
        else:
            freqs, gain = self._formula(theta, scaling, factor, original_length, beta_fast, beta_slow)
        self.frequencies = tuple(freqs)
        self.attention_factor = gain if attention_factor is None else _number("attention_factor", attention_factor)
        packed = _lib.Rotary(pairs=self.rotary_dim // 2, interleaved=int(interleaved), factor=self.attention_factor)
        for i, f in enumerate(freqs):
            num, den = f.as_integer_ratio()
            packed.turns[i] = (num * _TURN // den >> 192) % 2 ** 64
        self._packed = ctypes.string_at(ctypes.byref(packed), ctypes.sizeof(packed))

    def _formula(self, theta, scaling, factor, original_length, beta_fast, beta_slow):
        rd = self.rotary_dim
        if scaling == "ntk":
            if rd == 2:
                raise ValueError("ntk scaling needs a rotary_dim of 4 or more: its only pair is the fastest and the slowest")
            theta *= factor ** (rd / (rd - 2))
        freqs = [theta ** (-2 * i / rd) for i in range(rd // 2)]
        if scaling == "linear":
            freqs = [f / factor for f in freqs]
        if scaling != "yarn":
            return freqs, 1.0
        if original_length is None:
            raise ValueError("yarn scaling needs original_length")
        length = _number("original_length", original_length)
        fast, slow = _number("beta_fast", beta_fast), _number("beta_slow", beta_slow)
        if theta <= 1.0 or fast < slow:
            raise ValueError("yarn scaling needs theta > 1 and beta_fast >= beta_slow")
        pair = lambda turns: rd * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rd - 1)
        blend = lambda i: min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        return [f / factor * blend(i) + f * (1 - blend(i)) for i, f in enumerate(freqs)], 0.1 * math.log(factor) + 1 if factor > 1 else 1.0

    def __repr__(self):
        return (f"Rotary(head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, interleaved={self.interleaved}, "
                f"attention_factor={self.attention_factor:g})")


def check_rotary(rotary, head_dim: int, *, optional: bool = False):
    """The packed rotation of a `Rotary` for heads of `head_dim` elements (None for None)."""
    if rotary is None and optional:
        return None
    if not isinstance(rotary, Rotary):
        raise TypeError(f"rotary must be a Rotary, got {type(rotary).__name__}")
    if rotary.head_dim != head_dim:
        raise ValueError(f"rotary is for head dimension {rotary.head_dim}, got {head_dim}")
    return rotary._packed


def check_plain_call() -> None:
    """Refuses the transformations that would take these operations for something else."""
    if torch._C._are_functorch_transforms_active():
        raise NotImplementedError("torch.func transforms are unsupported; differentiate with reverse mode instead")
    if torch.jit.is_tracing():
        raise NotImplementedError("torch.jit.trace is unsupported: it would record the result as a constant")


def check_heads(name: str, t, like=None) -> None:
    """A [B, H, N, D] tensor that the kernels (or, on the CPU, the plain route) take."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError("forward-mode AD is unsupported; differentiate with reverse mode instead")
    if t.ndim != 4:
        raise ValueError(f"{name} must have rank 4 [B, H, N, D], got shape {tuple(t.shape)}")
    if t.numel() == 0:
        raise ValueError(f"every dimension of {name} must be positive, got {tuple(t.shape)}")
    if t.dtype not in (_CUDA_DTYPES if t.is_cuda else _CPU_DTYPES):
        raise TypeError(f"{name} dtype must be one of {', '.join(map(str, _CUDA_DTYPES if t.is_cuda else _CPU_DTYPES))}; got {t.dtype}")
    if t.is_cuda and t.shape[3] not in _CUDA_HEAD_DIMS:
        raise ValueError(f"CUDA head dimension D must be one of {_CUDA_HEAD_DIMS}, got {t.shape[3]}")
    if like is not None:
        if t.device != like.device:
            raise ValueError(f"{name} must be on {like.device}, got {t.device}")
        if t.dtype != like.dtype:
            raise ValueError(f"{name} must have dtype {like.dtype}, got {t.dtype}")


def turn(x: torch.Tensor, positions: torch.Tensor, rotary: Rotary) -> torch.Tensor:
    """Plain route: x [..., H, N, D] turned to positions [..., N], angles in 64 bits, in fp32 or x's wider type."""
    rd, wide = rotary.rotary_dim, torch.promote_types(x.dtype, torch.float32)
    freqs = torch.tensor(rotary.frequencies, dtype=torch.float64, device=x.device)
    angle = positions.double().unsqueeze(-2).unsqueeze(-1) * freqs
    c, s = (rotary.attention_factor * angle.cos()).to(wide), (rotary.attention_factor * angle.sin()).to(wide)
    head = x[..., :rd].to(wide)
    if rotary.interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = head[..., : rd // 2], head[..., rd // 2:]
        head = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((head.to(x.dtype), x[..., rd:]), -1)


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, rotary: Rotary, *, positions: torch.Tensor | None = None, offset: int = 0):
    """q [B, H_Q, N, D] and k [B, H_KV, N, D] turned to their positions, as (q, k), contiguous; k may be None.

    Row n sits at position offset + n, or at positions[n] or positions[b, n] (int32 or int64, any values).  Differentiable
    any number of times with respect to q and k.  CUDA tensors must be fp16 or bf16 with D in {32, 64, 128}.
    """
    # The usual valid CUDA call is recognised natively; everything else takes the checks below.
    if isinstance(rotary, Rotary) and isinstance(q, torch.Tensor) and q.is_cuda and not torch._C._are_functorch_transforms_active():
        out = _native.load().try_rotate(q, k, rotary._packed, rotary.head_dim, positions, offset, ops._CHECK_STATUS)
        if out is not None:
            return out
    check_plain_call()
    check_heads("q", q)
    packed = check_rotary(rotary, q.shape[3])
    if k is not None:
        check_heads("k", k, q)
        if k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]:
            raise ValueError(f"q and k must share batch size, rows and head dimension, got q={tuple(q.shape)} k={tuple(k.shape)}")
    offset = _as_count("offset", offset)
    if offset >= 2 ** 62:
        raise ValueError(f"offset must be below 2**62, got {offset}")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be an int32 or int64 torch.Tensor")
        if offset:
            raise ValueError("positions are given: offset must be 0")
        if tuple(positions.shape) not in ((q.shape[2],), (q.shape[0], q.shape[2])):
            raise ValueError(f"positions must have shape [N] or [B, N] of q={tuple(q.shape)}, got {tuple(positions.shape)}")
        if positions.device != q.device:
            raise ValueError(f"positions must be on {q.device}, got {positions.device}")
    if q.is_cuda:
        return _native.load().rotate(q, k, packed, positions, offset, ops._CHECK_STATUS)
    if positions is None:
        positions = torch.arange(offset, offset + q.shape[2])
    return turn(q, positions, rotary), None if k is None else turn(k, positions, rotary)
