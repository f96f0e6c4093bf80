"""Greedy CTC and candidates of packed lines (crec_ctc_greedy_lines, crec_candidates_lines) where the rules
leave a NaN."""
from __future__ import annotations

import numpy as np
import pytest

import line_ref as R
from test_gpu_line_rules import Case, line_places, logits_of

pytestmark = pytest.mark.gpu

# classes: a row in a warp's registers, in a team's, a warp a row in chunks (lines of 16 frames and more), from memory
CLASSES = [100, 800, 1500, 2100, 17000]
# A probability against 64 bits: at most 512 roundings of 2^-24 in any of the kernels (a lane's chain of 80 adds
# at 17,000 classes, 10 joins, the terms' own errors, 5 for each time a base rises)
ROOM = 2.0 ** -15


@pytest.mark.parametrize("classes", CLASSES)
def test_a_nan_shows_in_its_characters_probability(classes):
    """A character held over many frames, one of which allows a NaN: NaN wherever that frame lies, in every
    step of the frames' joining, and the character after it as if there were none."""
    first, second, places = 150, 30, [0, 1, 30, 31, 32, 33, 96, 127, 128, 129, 149]
    at = (np.arange(len(places) + 2) * (first + second)).astype(np.int32)
    rng = np.random.default_rng(classes)
    z = rng.normal(0, 1, (at[-1], classes)).astype(np.float32)
    z[np.arange(len(z)), np.tile(np.repeat([7, 9], [first, second]), len(at) - 1)] += 14
    plain = R.greedy(z, at)
    for i, t in enumerate(places):  # (the last line has none)
        z[at[i] + t, 50] = np.nan
    counts, ids, starts, probs = (x.cpu().numpy() for x in Case(z, at, None).greedy())
    for i, (wid, wst, wpr) in enumerate(plain):
        a = at[i]
        assert counts[i] == 2 and wid == [7, 9] and wst == [0, first]
        assert ids[a:a + 2].tolist() == wid and starts[a:a + 2].tolist() == wst
        if i < len(places):
            assert np.isnan(probs[a]), places[i]
        else:
            assert abs(probs[a] - wpr[0]) <= ROOM
        assert abs(probs[a + 1] - wpr[1]) <= ROOM


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("classes", CLASSES)
@pytest.mark.parametrize("named", [0, 400])
def test_a_nan_with_nothing_left_beside_it(classes, half, named):
    """Frames whose classes are NaN or nothing: they are blanks, and no candidate is left.  `named`: so many
    classes in the lines' histories (more than 256 go another way)."""
    rng = np.random.default_rng(classes + half)
    lines = 36 if classes <= 1500 else 3  # (enough rows for a warp to take its rows alone)
    at = line_places(rng, [40] * lines)
    z = logits_of(rng, at[-1], classes, half)
    z[:, 0] = -20
    nothing = [0, 3, 4, 39, 45, 79, 80, 90, 119]
    for i, t in enumerate(nothing):
        z[t] = np.nan if i % 3 == 0 else -np.inf
        z[t, 0] = np.nan
    rules = None
    if named:
        ids = [rng.permutation(classes)[:named] for _ in range(lines)]
        rules = {"history": np.concatenate(ids).astype(np.int32), "repeat": np.full(lines, 1.25, np.float32),
                 "history_at": np.concatenate([[0], np.cumsum([len(i) for i in ids])]).astype(np.int32)}
    c = Case(z, at, rules)
    c.want[nothing, 1:] = -np.inf  # (a NaN wins nothing)
    c.want[nothing, 0] = 0
    want = R.greedy(c.want, at)
    counts, ids, starts, _ = (x.cpu().numpy() for x in c.greedy())
    for i, (wid, wst, _) in enumerate(want):
        assert counts[i] == len(wid)
        assert ids[at[i]:at[i] + counts[i]].tolist() == wid and starts[at[i]:at[i] + counts[i]].tolist() == wst
    ids, logp, blank = (x.cpu().numpy() for x in c.candidates(3))
    assert (ids[nothing] == -1).all() and np.isneginf(logp[nothing]).all() and np.isnan(blank[nothing]).all()
    assert (np.delete(ids, nothing, 0) > 0).all() and np.isfinite(np.delete(blank, nothing, 0)).all()
