"""How far the sums of exp(z - best) may be off in the two ways of greedy CTC and candidates of packed lines
that add more terms one after another than a row in registers: a warp a row in chunks, its sum
rescaled each time the row's maximum rises, and lines with more of a history than a list keeps.

Counted in roundings of 2^-24, relative to the sum (every term is positive):
  the adds that one term goes through: its accumulator's chain, then the joins;
  a term itself: ex2's error 2^-22 (4), and its argument (v - best) log2 e, off by a rounding of log2 e
  and one of the fused product, each 2^-24 of |v - best|, which a sum of C terms weighs by at
  most ln C on average (a term's weight p has |v - best| <= -ln p);
  a rescaling: ex2 (4) and the product (1), and the bases' difference rounded, 2^-24 of how far the base
  rose, together at most |v - best| for each term, so ln C again;
  the end: the best's own term (4) and the division (1)."""
from __future__ import annotations

import numpy as np
import pytest

import line_ref as R
from test_gpu_line_rules import Case, some_rules

pytestmark = pytest.mark.gpu


def chunk_of(half, aligned):
    """A warp's chunk of a long row (classes) and the lanes' part of it."""
    lane = (32 if half else 16) if aligned else 16
    return 32 * lane, lane


def long_room(classes, half, aligned, rises):
    chunk, lane = chunk_of(half, aligned)
    chain = -(-classes // chunk) * lane // 4 + 8  # four accumulators a lane; at most 8 entries a lane
    joins = 2 + 5 + 1  # the accumulators, the lanes, the blank
    return (chain + joins + 4 + 3 * np.log(classes + 1) + 5 * (rises + 1) + 5) * 2.0 ** -24


def slow_room(classes, warps):
    chain = -(-classes // (256 * warps)) * 16  # spans of 256 classes: 8 a lane, and as many entries
    joins = 10 + 1
    return (chain + joins + 4 + 2 * np.log(classes + 1) + 5) * 2.0 ** -24


def check(c, room, k=16):
    """Greedy's characters and probabilities, the candidates and their log-probabilities."""
    got = [x.cpu().numpy() for x in c.greedy()]
    counts, ids, starts, probs = got
    some = 0
    for i, (wid, wst, wpr) in enumerate(R.greedy(c.want, c.line_at)):
        a, n = c.line_at[i], counts[i]
        assert ids[a:a + n].tolist() == wid and starts[a:a + n].tolist() == wst
        assert np.all(np.abs(probs[a:a + n] - wpr) <= room * np.array(wpr))
        some += n
    assert some > 0
    ids, logp, blank = (x.cpu().numpy() for x in c.candidates(k))
    wid, wlp, wbl = R.candidates(c.want, k)
    assert np.array_equal(ids, wid)
    for a, b in ((logp, wlp), (blank, wbl)):
        fin = np.isfinite(b)
        # the differences and the logarithm round once each, relative to |z - best| + ln C at most
        near = room + 2.0 ** -24 * (2 * np.abs(b[fin]) + 4 * np.log(c.z.shape[1] + 1) + 1)
        assert np.array_equal(a[~fin], b[~fin].astype(np.float32)) and np.all(np.abs(a[fin] - b[fin]) <= near)


@pytest.mark.parametrize("rise", [0.05, 0.5, 4.0])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("classes,pitch", [(2100, 2104), (12000, 12000), (12000, 12001), (16384, 16384)])
def test_a_maximum_that_rises_in_every_chunk(classes, pitch, half, rise):
    aligned = pitch % 8 == 0
    chunk, _ = chunk_of(half, aligned)
    rng = np.random.default_rng(classes)
    at = np.array([0, 40, 60, 97], np.int32)
    z = rng.normal(0, 0.02, (97, classes)) + rise * (np.arange(classes) // chunk)
    z[np.arange(97), rng.integers(classes - 50, classes, 97)] += 1
    z = z.astype(np.float16 if half else np.float32)
    for rules in ({}, some_rules(rng, 3, classes, longest=200, parts=("history",))):
        c = Case(z, at, rules, pitch)
        tops = [c.want[:, k:k + chunk].max(1) for k in range(0, classes, chunk)]
        if not rules:
            assert all((a < b).all() for a, b in zip(tops[:-1], tops[1:]))
        check(c, long_room(classes, half, aligned, len(tops)))


@pytest.mark.parametrize("classes,lines,warps", [(600, 40, 1), (800, 40, 1), (12000, 2, 16)])
def test_histories_past_a_list(classes, lines, warps):
    rng = np.random.default_rng(classes)
    length = 37 if lines > 2 else 9
    at = (np.arange(lines + 1) * length).astype(np.int32)
    z = rng.normal(0, 0.5, (at[-1], classes)).astype(np.float32)
    ids = [rng.permutation(classes)[:classes * 3 // 4] for _ in range(lines)]
    rules = {"history": np.concatenate(ids).astype(np.int32), "frequency": np.full(lines, 0.125, np.float32),
             "history_at": np.concatenate([[0], np.cumsum([len(i) for i in ids])]).astype(np.int32)}
    check(Case(z, at, rules), slow_room(classes, warps))
