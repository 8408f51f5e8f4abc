"""Rotations' frequencies, and what the rotation of positions refuses before anything is launched."""

import contextlib
import ctypes
import math

import pytest
import torch

from ojasx_amd import _native as N
from ojasx_amd import rotary, serve_ops as S


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


@pytest.fixture
def library(monkeypatch):
    fake = _Library()
    monkeypatch.setattr(N, "lib", lambda: fake)
    monkeypatch.setattr(N, "require_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(N, "stream_handle", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return fake


def test_frequencies():
    f, gain = rotary.frequencies(8, 10000.0)
    assert gain == 1 and f == pytest.approx([1, 0.1, 0.01, 0.001], rel=1e-12)
    assert rotary.frequencies(8, 10000.0, {"kind": "linear", "factor": 4})[0] == pytest.approx(
        [v / 4 for v in f], rel=1e-12)
    # the fastest pair as it was, the slowest divided by the factor
    g = rotary.frequencies(8, 10000.0, {"kind": "base", "factor": 8})[0]
    assert g[0] == 1 and g[-1] == pytest.approx(f[-1] / 8, rel=1e-12)
    f = rotary.frequencies(128)[0]
    g, gain = rotary.frequencies(128, scaling={"kind": "ramp", "factor": 16, "length": 4096})
    assert gain == pytest.approx(0.1 * math.log(16) + 1)
    # 4096 positions are 2^16 / 16 / 2 pi: pairs up to 20 turn over 32 times, from 46 on under once
    lo = math.floor(128 * math.log(4096 / (2 * math.pi * 32)) / (2 * math.log(10000)))
    hi = math.ceil(128 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000)))
    assert (lo, hi) == (20, 46)
    assert g[:lo + 1] == f[:lo + 1] and g[hi:] == [v / 16 for v in f[hi:]]
    assert g[33] == pytest.approx(f[33] * 0.5 + f[33] / 16 * 0.5, rel=1e-12)
    g, gain = rotary.frequencies(128, scaling={"kind": "wavelength", "factor": 8, "length": 8192})
    assert gain == 1
    for a, b in zip(f, g):
        turns = 8192 * a / (2 * math.pi)
        assert b == pytest.approx(a if turns >= 4 else a / 8 if turns <= 1 else
                                  a / 8 + (a - a / 8) * (turns - 1) / 3, rel=1e-12)
    g, gain = rotary.frequencies(6, scaling={"kind": "list", "factors": [1, 2, 4], "gain": 1.5})
    assert gain == 1.5 and g == pytest.approx(
        [a / b for a, b in zip(rotary.frequencies(6)[0], (1, 2, 4))])
    assert rotary.frequencies(2, scaling={"kind": "base", "factor": 8})[0] == [1.0]


def test_rates_are_fractions_of_a_turn():
    quarter = math.pi / 2
    r = rotary.from_frequencies([quarter, -quarter, 2 * math.pi + quarter, 0.0], device="cpu")
    got = [v / 2.0 ** 64 for v in r.rates.tolist()]
    assert got == pytest.approx([0.25, -0.25, 0.25, 0.0], abs=1e-15)
    r = rotary.from_frequencies(torch.tensor([1.0, 0.5], dtype=torch.float64), 1.2, True, "cpu")
    assert r.gain == 1.2 and r.interleaved and r.rates.dtype == torch.int64
    assert r.rates.tolist() == pytest.approx([2 ** 64 / (2 * math.pi), 2 ** 64 / (4 * math.pi)])
    assert rotary.rotation(64, device="cpu").rates.numel() == 32


@pytest.mark.parametrize("args", [
    (7,), (0,), (8, 0.0), (8, math.inf), (8, 1e4, {"kind": "other", "factor": 2}), (8, 1e4, {}),
    (8, 1e4, {"kind": "linear"}), (8, 1e4, {"kind": "linear", "factor": -1}),
    (8, 1e4, {"kind": "linear", "factor": 2, "length": 3}), (8, 1e4, {"kind": "ramp", "factor": 2}),
    (8, 1e4, {"kind": "wavelength", "factor": 2, "length": 9, "low": 4, "high": 4}),
    (8, 1.0, {"kind": "ramp", "factor": 2, "length": 9}), (8, 0.5, {"kind": "ramp", "factor": 2, "length": 9}),
    (4, 1e4, {"kind": "base", "factor": 1e300}), (512, 1e-320),
    (8, 1e4, {"kind": "list", "factors": [1, 2, 3]}),
    (8, 1e4, {"kind": "list", "factors": [1, 2, 3, 0]})])
def test_frequencies_that_cannot_be(args):
    if len(args) == 3 and args[2] == {}:
        assert rotary.frequencies(*args) == rotary.frequencies(8)  # nothing to scale
        return
    with pytest.raises(RuntimeError):
        rotary.frequencies(*args)


def test_rotations_that_cannot_be():
    for args in (([],), ([math.nan],), ([1.0], math.inf)):
        with pytest.raises(RuntimeError):
            rotary.from_frequencies(*args, device="cpu")


def test_rotary_is_taken_and_refused(library):
    q, k = torch.zeros(2, 5, 6, 80, dtype=torch.bfloat16), torch.zeros(2, 5, 2, 80, dtype=torch.bfloat16)
    pos, rates = torch.zeros(2, 5, dtype=torch.int32), torch.ones(40, dtype=torch.int64)
    rest = (1.0, False, False)
    a, b = S.rotary(q, k, pos, rates, *rest)
    assert a.shape == q.shape and b.shape == k.shape
    S.rotary(q, None, pos[0].long(), rates[:7], *rest)
    S.rotary(q[0], k[0], pos[0], rates, *rest)
    S.rotary(q[:, :0], k[:, :0], pos[:, :0], rates, *rest)
    assert library.calls == ["ojx_rotary"] * 4
    for args in ((q, k.float(), pos, rates), (q.double(), k.double(), pos, rates), (q, k[:1], pos, rates),
                 (q, k[:, :4], pos, rates), (q, k[..., :60], pos, rates), (q, k[0], pos, rates),
                 (q[0, 0], None, pos, rates), (q, k, pos.float(), rates), (q, k, pos[:, :4], rates),
                 (q, k, pos[:1], rates), (q[0], k[0], pos, rates), (q, k, pos, rates.int()),
                 (q, k, pos, rates[None]), (q, k, pos, torch.ones(41, dtype=torch.int64)),
                 (q, k, pos, rates[:0]), (q, k, pos, rates[::2])):
        with pytest.raises(RuntimeError):
            S.rotary(*args, *rest)
    assert len(library.calls) == 4


def test_cpu_tensors_raise():
    r = rotary.rotation(8, device="cpu")
    with pytest.raises(RuntimeError, match="ROCm"):
        rotary.rotate(torch.zeros(3, 1, 8), torch.zeros(3, dtype=torch.int32), r)


def test_c_abi_rejects_bad_arguments_before_launch():
    lib = N.lib()
    P = 256  # never read: every call is refused or has nothing to do
    q = dict(x=P, y=P, x_batch=0, x_token=480, x_head=80, y_batch=0, y_token=480, y_head=80, heads=6)
    rot = dict(rates=P, pairs=40, positions=P, positions64=0, interleaved=0, gain=1.0, inverse=0)

    def call(q_change=None, rot_change=None, k_change=None, batches=1, tokens=3, d=80, dtype=2,
             no_q=False, no_rot=False):
        a = N.RotaryRows(**{**q, **(q_change or {})})
        b = N.RotaryRows(**{**q, **k_change}) if k_change is not None else None
        r = N.Rotation(**{**rot, **(rot_change or {})})
        return lib.ojx_rotary(None if no_q else ctypes.byref(a), ctypes.byref(b) if b else None, batches,
                              tokens, d, dtype, None if no_rot else ctypes.byref(r), 0, 1, None)

    assert call(no_q=True) == -1 and call(no_rot=True) == -1
    assert call(dtype=5) == -3 and call(d=0) == -2 and call(d=5000) == -2
    assert call(tokens=-1) == -1 and call(batches=-1) == -1
    assert call(batches=1 << 20, tokens=1 << 20) == -1
    for change, code in ((dict(pairs=0), -2), (dict(pairs=41), -2), (dict(gain=math.nan), -1),
                         (dict(rates=0), -1), (dict(positions=0), -1), (dict(rates=260), -2),
                         (dict(positions=258), -2), (dict(positions=260, positions64=1), -2)):
        assert call(rot_change=change) == code, change
    for change, code in ((dict(x=0), -1), (dict(y=0), -1), (dict(heads=-1), -1), (dict(heads=5000), -1),
                         (dict(x_head=-1), -1), (dict(y_token=-1), -1), (dict(x=257), -2)):
        assert call(q_change=change) == code, change
        assert call(k_change=change) == code, change
    assert call(tokens=0) == 0 and call(batches=0) == 0
