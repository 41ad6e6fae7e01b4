"""The oracle of the cache operators against properties that a mistake in it would break."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import cache as oc
from oracle import quant as oq


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_keeps_lengths_adds_angles_and_leaves_the_rest(interleaved):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 3, 32))
    f = 100.0 ** -(np.arange(8) / 8)
    pos = np.array([0, 1, 7, 1000, -3])
    y = oc.rotate(x, pos, f, interleaved)
    assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 16:], x[..., 16:])
    np.testing.assert_allclose((y**2).sum(-1), (x**2).sum(-1), rtol=1e-13)
    np.testing.assert_allclose(oc.rotate(y, 5 - pos, f, interleaved), oc.rotate(x, 0 * pos + 5, f, interleaved), atol=1e-10)
    pair = (0, 1) if interleaved else (0, 8)  # frequency 1: the position is the angle
    assert y[1, 0, pair[0]] == pytest.approx(x[1, 0, pair[0]] * np.cos(1) - x[1, 0, pair[1]] * np.sin(1))
    np.testing.assert_allclose(oc.rotate(x, pos, f, interleaved, 2.0)[..., :16], 2 * y[..., :16])


def test_quantize_is_the_group_quantizer_and_marks_what_is_not_finite():
    x = torch.randn((6, 128), generator=torch.Generator().manual_seed(1)).bfloat16().float().numpy()
    x[3] = 0
    codes, scales = oc.quantize(x)
    want, s = oq.per_group_quant_fp8(x)
    assert np.array_equal(codes, want) and np.array_equal(scales, s[0])
    x[1, 5], x[2, 0] = np.nan, -np.inf
    codes, scales = oc.quantize(x)
    assert not codes[1:3].any() and np.isnan(scales[1:3]).all() and np.array_equal(codes[4:], want[4:])


def test_e4m3_table_is_torchs():
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(oc.E4M3, want, equal_nan=True)


def test_attention_against_one_softmax_over_everything():
    rng = np.random.default_rng(2)
    codes = [rng.integers(0, 120, (4, 2, 16, 64)).astype(np.uint8) for _ in "kv"]
    scales = [rng.random((4, 2, 16)).astype(np.float32) * 0.05 for _ in "kv"]
    table = np.array([[2, 0], [3, 9]], dtype=np.int32)  # page 9 is none
    q = rng.standard_normal((4, 4, 64)) * 0.3
    mask = np.array([[1, 0, 0], [0, 0, 0], [1, 0, 1], [1, 1, 0]], dtype=bool)
    out, lse, weighed, _ = oc.attention(q, *codes, *scales, table, [21, 17], [0, 3, 4], mask, 0.125)
    k = np.concatenate([oc.E4M3[codes[0][p]] * scales[0][p][..., None] for p in (2, 0)], 1)[:, :21]
    v = np.concatenate([oc.E4M3[codes[1][p]] * scales[1][p][..., None] for p in (2, 0)], 1)[:, :21]
    keep = np.r_[np.ones(18, bool), [True, False, True]]
    w = np.exp(q[2, 3] @ k[1].T * 0.125) * keep
    np.testing.assert_allclose(out[2, 3], w @ v[1] / w.sum(), rtol=1e-12)
    assert lse[2, 3] == pytest.approx(np.log(w.sum()))
    # the second sequence: its token is position 16, on the page that is none, so it sees the 16 of page 3
    k1, v1 = (oc.E4M3[codes[i][3, 0]] * scales[i][3, 0][:, None] for i in (0, 1))
    w = np.exp(q[3, 1] @ k1.T * 0.125)
    np.testing.assert_allclose(out[3, 1], w @ v1 / w.sum(), rtol=1e-12)
    none, at, *_ = oc.attention(q[:1], *codes, *scales, table[:1], [1], [0, 1], np.zeros((1, 1), bool), 1.0)
    assert not none.any() and (at == -np.inf).all()
    assert (weighed >= np.abs(out) - 1e-12).all()
