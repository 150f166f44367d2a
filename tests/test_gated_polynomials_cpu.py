"""The polynomials of the gated kernels meet the errors that stand beside them: their coefficients, read
from the sources, against the functions in 64 bits (rounding while they are evaluated comes on top)."""
from __future__ import annotations

import math
import re
from pathlib import Path

import numpy as np

CSRC = Path(__file__).resolve().parent.parent / "semambaxlinoss_b200" / "csrc"
NUMBER = r"-?\d+\.\d+(?:e-?\d+)?"


def _body(file, name):
    text = (CSRC / file).read_text()
    start = text.index(f" {name}(")
    return text[start:text.index("\n}", start)]


def _horner3(file, name):
    found = re.search(rf"horner3\(m, ({NUMBER})f, ({NUMBER})f, ({NUMBER})f, ({NUMBER})f\)", _body(file, name))
    return [float(np.float32(c)) for c in found.groups()]


def _value(c, v):
    out = np.zeros_like(v)
    for k in reversed(c):
        out = out * v + k
    return out


def test_decay_and_root_near_one():
    m = np.linspace(0, 0.125, 20001)[1:]
    decay = 1 + m * _value(_horner3("gated_lru.cu", "decay_near"), m)
    assert np.abs(decay / np.exp(-m) - 1).max() <= 3.7e-9
    root = np.sqrt(-np.expm1(-2 * m) / (2 * m))
    off = _value(_horner3("gated_lru.cu", "root_near"), m) / root - 1
    assert off.max() <= 3.1e-8 and off.min() >= -3.1e-8


def test_normal_tail():
    numbers = re.findall(rf"({NUMBER})f", _body("gated_mlp.cu", "normal_tail"))
    c = [float(np.float32(v)) for v in numbers if v not in ("0.35355339059327379", "1.", "-0.72134752044448170")]
    assert len(c) == 9
    z = np.linspace(0, 9.5, 20001)
    t = 1 / (1 + z / 2)
    tail = t * _value(c[::-1], t) * np.exp(-z * z)
    off = tail / np.array([math.erfc(v) / 2 for v in z]) - 1
    assert np.abs(off).max() <= 6.6e-8
    # The exponential's argument -g^2 / 2 as the kernel forms it, in fp32: what its roundings do to the tail.
    g = np.linspace(0, 13, 20001).astype(np.float32)
    arg = (np.float32(-0.72134752044448170) * g) * g
    off = np.exp2(arg.astype(np.float64)) / np.exp(-g.astype(np.float64) ** 2 / 2) - 1
    assert np.abs(off).max() <= 1.1e-5 and np.abs(off[g < 3]).max() <= 6e-7
