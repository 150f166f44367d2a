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
