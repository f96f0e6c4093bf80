"""The head with adapters (crec_adapters_logits) where its values are not ordinary: NaN and infinities in
features, adapters and scales show where the formula has them and nowhere else, and inner sums
that need more than one tf32 word keep every bit of it."""
from __future__ import annotations

import numpy as np
import pytest

from carbon_rec import native
from test_gpu_adapters import Case

pytestmark = pytest.mark.gpu

LENGTHS = [9, 30, 1, 40, 20, 17, 33]


def formula(c):
    """The logits in 64 bits by plain sums (every product of an infinity or a NaN in them), and what
    roundings are relative to, as the other adapter tests count it."""
    with np.errstate(all="ignore"):
        x, w, b = c.x.astype(np.float64), c.w.astype(np.float64), c.b.astype(np.float64)
        z = np.einsum("fk,ck->fc", x, w) + b
        mag = np.einsum("fk,ck->fc", abs(x), abs(w)) + abs(b)
        for i, a in enumerate(c.adapter):
            if 0 <= a < len(c.sets):
                A, B, s = c.sets[a]
                A, B, s = A.astype(np.float64), B.astype(np.float64), np.float64(np.float32(s))
                rows = slice(c.line_at[i], c.line_at[i + 1])
                z[rows] += np.einsum("fj,cj->fc", s * np.einsum("fk,jk->fj", x[rows], A), B)
                mag[rows] += abs(s) * np.einsum("fj,cj->fc", np.einsum("fk,jk->fj", abs(x[rows]), abs(A)), abs(B))
    return z, mag


def check_values(c, half=False):
    import torch
    c.upload()
    h = c.open()
    out = c.queue(h, half)
    torch.cuda.synchronize()
    h.close()
    got = out.cpu().numpy().reshape(c.rows, c.classes).astype(np.float64)
    want, mag = formula(c)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    far = np.isinf(want)
    assert np.array_equal(got[far], want[far])
    fin = np.isfinite(want)
    rank = max(a.shape[0] for a, _, _ in c.sets)
    room = (2 * c.k + 2 * rank + 8) * 2.0 ** -23 * mag[fin]
    if half:
        room = room + 2.0 ** -11 * np.abs(want[fin]) + 2.0 ** -25
    assert np.all(np.abs(got[fin] - want[fin]) <= room)
    return want


def a_nan(c, own):
    c.sets[1][0][own - 1, 3] = np.nan


def a_infinity(c, own):
    c.sets[1][0][0, 3] = np.inf


def b_nan(c, own):
    c.sets[1][1][5, own - 1] = np.nan


def scale_nan(c, own):
    c.sets[1] = (*c.sets[1][:2], float("nan"))


def scale_infinity(c, own):
    c.sets[1] = (*c.sets[1][:2], float("inf"))


def x_nan(c, own):
    c.x[c.line_at[1] + 2, 7] = np.nan


def x_infinity(c, own):
    """With all weights of its channel positive, every logit is an infinity of the formula, none NaN."""
    c.x[c.line_at[1] + 2, 7] = np.inf
    c.w[:, 7] = 0.05
    c.sets[1][0][:, 7] = 0.02
    c.sets[1][1][:] = np.abs(c.sets[1][1]) + np.float16(0.01)


def inner_infinities(c, own):
    """An inner sum of infinity less infinity."""
    c.sets[1][0][0, 3] = np.inf
    c.sets[1][0][0, 4] = -np.inf
    c.x[:, 3:5] = 1


SPOILED = [a_nan, a_infinity, b_nan, scale_nan, scale_infinity, x_nan, x_infinity, inner_infinities]


@pytest.mark.parametrize("spoil", SPOILED)
@pytest.mark.parametrize("rank,own", [(8, 1), (16, 11), (32, 32), (32, 17), (64, 40)])
def test_nan_and_infinities_show_in_their_own_lines(rank, own, spoil):
    """Lines of the spoiled adapter beside lines of a sound one and of none, in one tile and in tiles of few
    frames; `own` of the spoiled one's rows of the handle's `rank` are its own."""
    for lengths in (LENGTHS, [1] * 90):
        c = Case(72, 100, [rank, own, 1], lengths, seed=rank)
        c.adapter = np.array([0, 1, -1, 1, 2, 0, 1] * 13, np.int32)[:len(lengths)]
        c.sets[1][0][c.sets[1][0] == 0] = 0.01  # (an infinity times 0 is NaN)
        spoil(c, own)
        want = check_values(c)
        bad = ~np.isfinite(want).all(1)
        assert bad.any() and not bad[:c.line_at[1]].any()


@pytest.mark.parametrize("spoil", [a_nan, scale_infinity, x_infinity])
def test_nan_and_infinities_in_float16(spoil):
    c = Case(256, 800, [16, 4, 1], LENGTHS)
    c.adapter = np.array([0, 1, -1, 1, 2, 0, 1], np.int32)
    c.sets[1][0][c.sets[1][0] == 0] = 0.01
    spoil(c, 4)
    check_values(c, True)


def test_inner_sums_up_to_the_largest_float():
    """An inner sum within half a unit of a tf32 word of the largest float stays finite."""
    for scale in (0x7f7fffff, 0x7f7ff000, 0x7f7fefff, 0xff7fffff, 0xff7ff001):
        c = Case(16, 40, [1], [70], seed=3)
        c.adapter = np.zeros(1, np.int32)
        c.w[:] = 0
        c.b[:] = 0
        c.x[:] = 0
        c.x[:, 2] = 1
        s = float(np.array([scale], np.uint32).view(np.float32)[0])
        c.sets = [(np.eye(1, 16, 2, dtype=np.float16), np.full((40, 1), 2.0 ** -14, np.float16), s)]
        want = check_values(c)
        assert np.isfinite(want).all()
