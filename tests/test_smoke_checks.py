"""What the smoke check of a gated step lets pass, and what not."""

import numpy as np
import pytest

from __graft_entry__ import _check_gated_step
from oracle import fp8_oracle as fo


def bf16(v):
    bits = v.astype(np.float32).view(np.uint32)
    return ((bits + 0x7fff + (bits >> 16 & 1)) & 0xffff0000).astype(np.uint32).view(np.float32).astype(np.float64)


def step(n=20, f=48, k=144):
    rng = np.random.default_rng(n)
    x, dh = bf16(rng.standard_normal((n, k))), bf16(rng.standard_normal((n, f)))
    w = fo.numbers(rng.standard_normal((2 * f, k)) * k ** -0.5, "square")
    want = fo.numbers(x, "row") @ w.T
    z, h = bf16(want), bf16(fo.activation(want[:, :f], "silu")[0] * want[:, f:])
    value, slope = fo.activation(z[:, :f], "silu")
    dz = np.concatenate((dh * z[:, f:] * slope, dh * value), 1)
    return {"x": x, "w": w, "dh": dh, "z": z, "h": h, "dx": fo.numbers(dz, "row") @ w, "dw": fo.numbers(dz, "column").T @ fo.numbers(x, "column")}


@pytest.mark.parametrize("n", [1, 16, 300])
def test_a_right_step_passes(n):
    _check_gated_step(**step(n))


def halves(v):
    return np.concatenate((v[:, v.shape[1] // 2:], v[:, :v.shape[1] // 2]), 1)


def sloped(s):
    """dx of a slope that leaves out the activation's second term."""
    f = s["h"].shape[1]
    g, u = s["z"][:, :f], s["z"][:, f:]
    sigma = 1 / (1 + np.exp(-g))
    dz = np.concatenate((s["dh"] * u * sigma, s["dh"] * g * sigma), 1)
    return fo.numbers(dz, "row") @ s["w"]


@pytest.mark.parametrize("name,wrong", [("z", lambda s: halves(s["z"])), ("z", lambda s: s["z"] * (1 + 2.0 ** -7)), ("h", lambda s: s["h"] * 0.98), ("h", lambda s: np.roll(s["h"], 1, 1)), ("dx", sloped),
                                        ("dx", lambda s: np.zeros_like(s["dx"])), ("dw", lambda s: np.roll(s["dw"], s["dw"].shape[0] // 2, 0)), ("dw", lambda s: np.full_like(s["dw"], np.nan))])
def test_a_wrong_one_does_not(name, wrong):
    s = step()
    s[name] = wrong(s)
    with pytest.raises(AssertionError, match=name):
        _check_gated_step(**s)
