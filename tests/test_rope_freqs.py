"""mako_rope_freqs (host code) against its formulas."""
import math

import numpy as np
import pytest


def test_scalings():
    import mako_attn as M
    rot, theta = 128, 10000.0
    i = np.arange(rot // 2)
    f = theta ** (-2.0 * i / rot)
    # pow is within a few units in the last place of 64 bits
    close = dict(rtol=1e-14, atol=0)
    np.testing.assert_allclose(M.rope_freqs(rot, theta), f, **close)
    np.testing.assert_allclose(M.rope_freqs(rot, theta, M.ROPE_LINEAR, 4.0), f / 4, **close)
    base = M.rope_freqs(rot, theta, M.ROPE_BASE, 8.0)
    assert base[0] == 1.0 and math.isclose(base[-1], f[-1] / 8, rel_tol=1e-13)
    assert (np.diff(f / base) > 0).all()
    parts = M.rope_freqs(rot, theta, M.ROPE_PARTS, 4.0, 8192.0, 1.0, 32.0)
    turns = 8192.0 * f / (2 * math.pi)
    np.testing.assert_allclose(parts[turns >= 32], f[turns >= 32], **close)
    np.testing.assert_allclose(parts[turns <= 1], f[turns <= 1] / 4, **close)
    mid = (turns > 1) & (turns < 32)
    g = (turns[mid] - 1) / 31
    assert mid.any()
    np.testing.assert_allclose(parts[mid], f[mid] * (g + (1 - g) / 4), rtol=1e-13)
    assert M.rope_freqs(2, theta).tolist() == [1.0]


def test_refusals():
    import mako_attn as M
    for args, text in [((0, 1e4), "0 rotated"), ((7, 1e4), "7 rotated"), ((258, 1e4), "258 rotated"),
                       ((2, 1e4, M.ROPE_BASE, 2.0), "2 rotated"), ((64, 1.0), "theta"), ((64, math.nan), "theta"),
                       ((64, 1e4, 4), "scaling 4"), ((64, 1e4, -1), "scaling -1"),
                       ((64, 1e4, M.ROPE_LINEAR, 0.5), "factor"), ((64, 1e4, M.ROPE_LINEAR, math.nan), "factor"),
                       ((64, 1e4, M.ROPE_PARTS, 2.0, 0.0, 1.0, 2.0), "context"),
                       ((64, 1e4, M.ROPE_PARTS, 2.0, 64.0, 2.0, 2.0), "low 2")]:
        with pytest.raises(M.MakoError, match=text):
            M.rope_freqs(*args)
    import ctypes
    assert M.lib().mako_rope_freqs(64, 1e4, 0, 1.0, 0.0, 0.0, 0.0, None) == M.EINVAL
    assert ctypes.string_at(M.lib().mako_attn_last_error()) == b"rope_freqs: null freq"
