"""The head with adapters: inner sums of more bits than one tf32 word holds reach the logits whole.

The head's own weights and biases are 0, features and A whole numbers, the scale a power of 2, and each
class takes one inner sum (B one power of 2 a class), so a logit is B h with h = scale * sum_k x_k A_jk
exact in float32.  Two tf32 words of 11 significant bits each hold h to 2^-23 of it (exactly to 22 bits);
their two products are exact, and their sum in float32 is off by a unit of 2^-23 at most.  So the
logits are within 2^-22 of B h, where one word alone would be off by up to 2^-11."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_adapters import Case

LENGTHS = [62, 0, 1, 7, 128, 129, 3]
ROOM = 2.0 ** -22
# padded ranks 8, 16, 32 and 64; ranks of their own on either side of the 16 and 32 columns that are copied at once
RANKS = [[8, 5, 1], [16, 9, 3], [32, 17, 31], [64, 33, 48], [64, 64, 32]]


def whole_numbers(k, classes, ranks, scale):
    c = Case(k, classes, ranks, LENGTHS, seed=sum(ranks))
    rng = np.random.default_rng(k)
    c.adapter = np.array([0, 1, 2, -1, 1, 0, 2], np.int32)
    c.w[:] = 0
    c.b[:] = 0
    c.x[:] = rng.integers(-255, 256, c.x.shape)
    sets = []
    for r in ranks:
        B = np.zeros((classes, r), np.float16)
        B[np.arange(classes), np.arange(classes) % r] = 2.0 ** rng.integers(-8, 1, classes)
        sets.append((rng.integers(-63, 64, (r, k)).astype(np.float16), B, scale))
    c.sets = sets
    return c


def inner(c, i):
    """h of line i and the class's place in it, exactly."""
    A, B, s = c.sets[c.adapter[i]]
    rows = slice(c.line_at[i], c.line_at[i + 1])
    h = (c.x[rows].astype(np.int64) @ A.astype(np.int64).T) * s
    return h, np.arange(c.classes) % A.shape[0], B[np.arange(c.classes), np.arange(c.classes) % A.shape[0]].astype(np.float64)


def expected(c, word=lambda h: h):
    z = np.zeros((c.rows, c.classes))
    for i, a in enumerate(c.adapter):
        if a >= 0:
            h, j, b = inner(c, i)
            z[c.line_at[i]:c.line_at[i + 1]] = word(h)[:, j] * b
    return z


def one_word(h):
    """h as a single tf32 word, rounded."""
    b = (h.astype(np.float32).view(np.uint32) + 0x1000) & 0xffffe000
    return b.view(np.float32).astype(np.float64)


def near(got, want):
    return bool(np.all(np.abs(got - want) <= ROOM * np.abs(want)))


@pytest.mark.parametrize("ranks", RANKS)
@pytest.mark.parametrize("k", [8, 72, 512])
def test_the_cases_tell_one_word_from_two(ranks, k):
    """On the CPU: inner sums are exact in float32, reach past float16 where scaled, and logits made of one
    word of them, or of the low words a block of 32 columns off, are outside the room."""
    c = whole_numbers(k, 130, ranks, 16.0)
    for i in (0, 1, 2, 4, 5, 6):
        h, _, _ = inner(c, i)
        assert np.abs(h).max(initial=0) < 16 * 2 ** 24
    assert np.abs(inner(c, 5)[0]).max() > 65504
    want = expected(c)
    assert near(want, want) and not near(expected(c, one_word), want)

    def low_words_elsewhere(h):
        hi = one_word(h)
        return hi + np.roll(h - hi, 1, axis=1)
    if min(ranks) > 1:
        assert not near(expected(c, low_words_elsewhere), want)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 16.0])
@pytest.mark.parametrize("ranks", RANKS)
@pytest.mark.parametrize("k", [8, 72, 512])
def test_inner_sums_keep_their_bits(ranks, k, scale):
    import torch
    c = whole_numbers(k, 130, ranks, scale)
    c.upload()
    h = c.open()
    out = c.queue(h)
    torch.cuda.synchronize()
    h.close()
    assert near(out.cpu().numpy().reshape(c.rows, c.classes).astype(np.float64), expected(c))


# (k, classes, ranks, lengths, the lines' adapters): the largest class count, ranks of either half of the
# columns, tiles of few frames
EVERY = [(64, 12000, [32] * 3, [40, 90], [2, 0]), (192, 1500, [4, 64, 1, 33], LENGTHS, [1, 0, 3, 2, 1, 3, 0]),
         (512, 801, [64, 64, 5], LENGTHS, [0, 1, 2, 0, 1, 1, 2]), (256, 800, [16, 8, 32], [1] * 70, [0, 1, 2, 1, 0] * 14)]


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("k,classes,ranks,lengths,adapter", EVERY)
def test_every_line_has_an_adapter(k, classes, ranks, lengths, adapter, half):
    c = Case(k, classes, ranks, lengths)
    c.adapter = np.array(adapter, np.int32)
    assert (c.adapter >= 0).all() and (c.adapter < len(ranks)).all()
    c.upload()
    h = c.open()
    c.check(c.queue(h, half), half)
    h.close()
