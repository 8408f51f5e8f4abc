"""Rotated positions: queries and keys turned pair by pair by an angle that grows with the position.

    r = rotary.rotation(head_dim, base=10000.0, device="cuda")      # once for a model
    q, k = rotary.rotate_qk(q, k, positions, r)                      # [..., heads, head size]

A head's first ``2 * pairs`` elements are pairs, ``(i, i + pairs)`` or interleaved ``(2i, 2i + 1)``;
the rest of the head is copied.  Angles come from whole-number products modulo a turn, so they are
as good at position 10 million as at 10, and no table is kept.  ``kv8.rotate_append`` does the same
on the way into the cache.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _native as N
from . import serve_ops as S


class Rotation(NamedTuple):
    """What turns a head's pairs (``rotation`` makes it)."""

    rates: torch.Tensor        # int64 [pairs]: turns per position in units of 2^-64
    gain: float = 1.0          # factor of the rotated elements
    interleaved: bool = False  # pairs (2i, 2i + 1), else (i, i + pairs)


def _number(scaling: dict, name: str, default: Optional[float] = None) -> float:
    v = scaling.pop(name, default)
    if v is None:
        raise RuntimeError(f"scaling {scaling!r} lacks {name!r}")
    v = float(v)
    if not math.isfinite(v) or v <= 0:
        raise RuntimeError(f"scaling's {name} is {v}, expected a positive number")
    return v


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None
                ) -> Tuple[Sequence[float], float]:
    """(radians per position of each pair, gain): ``base ** (-2 i / rotary_dim)``, scaled for
    contexts longer than a model was trained with.  ``scaling`` is one of

    * ``{"kind": "linear", "factor": s}``: all divided by s;
    * ``{"kind": "base", "factor": s}``: the base times ``s ** (rotary_dim / (rotary_dim - 2))``,
      which keeps the fastest pair and divides the slowest by s;
    * ``{"kind": "ramp", "factor": s, "length": n, "fast": 32, "slow": 1, "gain": 0.1 ln s + 1}``:
      pairs that turn over ``fast`` times in the n positions of training stay, those under ``slow``
      are divided by s, between them a line over the pairs' numbers (Peng et al., 2023);
    * ``{"kind": "wavelength", "factor": s, "length": n, "low": 1, "high": 4}``: the same by turns in
      n positions, over ``high`` stay, under ``low`` are divided, a line over the turns between;
    * ``{"kind": "list", "factors": [...], "gain": 1}``: each pair divided by its own.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise RuntimeError(f"rotary_dim must be even and positive (got {rotary_dim})")
    if not (math.isfinite(base) and base > 0):
        raise RuntimeError(f"base is {base}, expected a positive number")
    n, gain = rotary_dim // 2, 1.0
    rest = dict(scaling or {"kind": None})
    kind = rest.pop("kind", "")
    s = _number(rest, "factor") if kind in ("linear", "base", "ramp", "wavelength") else 1.0
    try:
        b = base * s ** (rotary_dim / (rotary_dim - 2)) if kind == "base" and n > 1 else base
        f = [b ** (-2 * i / rotary_dim) for i in range(n)]
    except OverflowError:
        raise RuntimeError(f"base {base} with scaling {scaling!r} passes float64's range") from None
    if kind == "linear":
        f = [v / s for v in f]
    elif kind == "ramp":
        if not base > 1:
            raise RuntimeError(f"base is {base}, expected over 1 for a ramp over slower pairs")
        length, fast, slow = (_number(rest, *a) for a in (("length",), ("fast", 32), ("slow", 1)))
        gain = _number(rest, "gain", 0.1 * math.log(s) + 1 if s > 1 else 1.0)
        lo, hi = (rotary_dim * math.log(length / (2 * math.pi * t)) / (2 * math.log(base))
                  for t in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rotary_dim - 1)
        for i in range(n):
            t = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            f[i] = f[i] / s * t + f[i] * (1 - t)
    elif kind == "wavelength":
        length, low, high = (_number(rest, *a) for a in (("length",), ("low", 1), ("high", 4)))
        if not high > low:
            raise RuntimeError(f"scaling's high is {high}, expected over its low, {low}")
        for i in range(n):
            t = min(max((length * f[i] / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f[i] = (1 - t) * f[i] / s + t * f[i]
    elif kind == "list":
        factors = [float(v) for v in rest.pop("factors", ())]
        if len(factors) != n or not all(math.isfinite(v) and v > 0 for v in factors):
            raise RuntimeError(f"scaling's factors are {factors}, expected {n} positive numbers")
        gain = _number(rest, "gain", 1.0)
        f = [v / w for v, w in zip(f, factors)]
    elif kind not in (None, "base"):
        raise RuntimeError(f"unknown scaling {scaling!r}")
    if rest:
        raise RuntimeError(f"scaling of kind {kind!r} takes no {sorted(rest)}")
    return f, gain


def from_frequencies(freqs: Union[torch.Tensor, Sequence[float]], gain: float = 1.0,
                     interleaved: bool = False,
                     device: Union[str, torch.device, None] = "cuda") -> Rotation:
    """A rotation by given radians per position, one for each pair."""
    if isinstance(freqs, torch.Tensor):
        freqs = freqs.detach().double().cpu().flatten().tolist()
    rates = []
    for f in freqs:
        turns = float(f) / (2 * math.pi)
        if not math.isfinite(turns):
            raise RuntimeError(f"a frequency is {f}")
        # the fraction of a turn as a whole number of 2^-64, wrapped into int64's range
        r = round(math.fmod(turns, 1.0) * 2.0 ** 64) % (1 << 64)
        rates.append(r - (1 << 64) if r >> 63 else r)
    if not rates:
        raise RuntimeError("a rotation needs a pair")
    if not math.isfinite(gain):
        raise RuntimeError(f"gain is {gain}")
    return Rotation(torch.tensor(rates, dtype=torch.int64, device=device), float(gain),
                    bool(interleaved))


def rotation(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[dict] = None,
             interleaved: bool = False,
             device: Union[str, torch.device, None] = "cuda") -> Rotation:
    """The rotation of a head's first ``rotary_dim`` elements; ``frequencies`` has the scalings."""
    f, gain = frequencies(rotary_dim, base, scaling)
    return from_frequencies(f, gain, interleaved, device)


def _call(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, r: Rotation):
    args = (q, k, positions, r.rates, r.gain, r.interleaved, False)
    if not torch.compiler.is_compiling():
        e = N.eager()  # None: with a gradient to record; not plain eager work at all
        out = e.rotary(*args) or e.rotary_recorded(*args)
        if out is not None:
            return out
    return S.rotary(*args)


def rotate(x: torch.Tensor, positions: torch.Tensor, rotation: Rotation) -> torch.Tensor:
    """``x [tokens, heads, head size]`` or ``[batch, tokens, heads, head size]`` with the heads'
    pairs turned; ``positions`` (int32 or int64, any sign) are of x's leading sizes, or ``[tokens]``
    for every batch alike.  A view with any strides over batch, tokens and heads is taken as it
    lies.  Gradients pass to ``x``, any number of times."""
    return _call(x, None, positions, rotation)[0]


def rotate_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotation: Rotation
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rotate`` of queries and keys (other numbers of heads, the same head size) in one launch."""
    out = _call(q, k, positions, rotation)
    return out[0], out[1]
