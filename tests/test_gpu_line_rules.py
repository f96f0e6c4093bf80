"""The calls on packed lines' logits under rules (crec_logit_rules, crec_ctc_greedy_lines,
crec_candidates_lines) against the definition restated in numpy (line_ref.py): ruled logits, ids,
counts and starts exactly; probabilities within a float32 sum's rounding of 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import line_ref as R
from carbon_rec import native

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()


def some_rules(rng, lines, classes, longest=40, parts=("history", "bias", "allowed")):
    """Rules with everything in them that can go wrong: empty histories, ids outside the classes, indexes of no
    table and no set, a set that leaves nothing, a bias of -inf, repeated ids."""
    r = {}
    if "history" in parts:
        n = rng.integers(0, longest + 1, lines)
        r["history_at"] = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        ids = (classes * rng.random(max(1, n.sum())) ** 3).astype(np.int32)
        ids[rng.random(len(ids)) < 0.05] = classes + 3
        ids[rng.random(len(ids)) < 0.05] = -1
        r["history"] = ids
        r["repeat"] = rng.uniform(0.8, 1.6, lines).astype(np.float32)
        r["presence"] = rng.uniform(0, 0.6, lines).astype(np.float32)
        r["frequency"] = rng.uniform(0, 0.3, lines).astype(np.float32)
    if "bias" in parts:
        r["bias"] = rng.normal(0, 1, (3, classes)).astype(np.float32)
        r["bias"][1, rng.random(classes) < 0.2] = -np.inf
        r["bias_of"] = rng.integers(-1, 4, lines).astype(np.int32)  # 3: no table
    if "allowed" in parts:
        words = (classes + 31) // 32
        bits = rng.random((5, words * 32)) < np.linspace(0.05, 1, 5)[:, None]
        bits[:, 0] = True
        bits[1] = False  # leaves nothing
        bits[3, 0] = False  # no blank
        r["allowed"] = (bits.reshape(5, words, 32) * (1 << np.arange(32, dtype=np.uint64))).sum(2).astype(np.uint32)
        r["set_of"] = rng.integers(-1, 6, lines).astype(np.int32)  # 5: no set
    return r


def line_places(rng, lengths, first=0):
    return np.concatenate([[first], first + np.cumsum(lengths)]).astype(np.int32)


def logits_of(rng, rows, classes, half, grid=False):
    z = rng.normal(0, 2, (rows, classes))
    z[:, 0] += np.where(rng.random(rows) < 0.5, 6, 0)
    say = np.repeat(rng.integers(0, classes, rows // 3 + 1), 3)[:rows]  # a character's frames side by side
    z[np.arange(rows), say] += 5 * rng.random(rows)
    if grid:  # many ties
        z = np.rint(z * 2) / 2
    return z.astype(np.float16 if half else np.float32)


class Case:
    """Logits in rows of `pitch` (the array `skip` elements into its memory), lines and rules on the GPU."""

    def __init__(self, z, line_at, rules, pitch=None, skip=0):
        import torch
        rows, classes = z.shape
        pitch = pitch or classes
        self.z, self.line_at, self.rules = z, line_at, rules
        flat = np.full(skip + rows * pitch, 77, z.dtype)
        flat[skip:].reshape(rows, pitch)[:, :classes] = z
        self.keep = [dev(flat), dev(line_at)]
        self.kind = native.FP16 if z.dtype == np.float16 else native.FP32
        self.frames = native.LineLogits(self.keep[0].data_ptr() + skip * z.dtype.itemsize, self.kind, classes, pitch, rows,
                                        len(line_at) - 1, self.keep[1].data_ptr())
        self.crules = None
        if rules:
            d = {k: dev(v) for k, v in rules.items()}
            self.keep.append(d)
            self.crules = native.Rules(biases=len(rules.get("bias", ())), sets=len(rules.get("allowed", ())),
                                       **{k: v.data_ptr() for k, v in d.items()})
        self.want = R.ruled(z, line_at, rules or {})
        self.torch = torch

    def ruled(self, out_half=False, pitch=None, skip=0, stream=0):
        rows, classes = self.z.shape
        pitch = pitch or classes
        t = self.torch.float16 if out_half else self.torch.float32
        out = self.torch.full((skip + rows * pitch,), 55.0, dtype=t, device="cuda")
        native.logit_rules(self.frames, self.crules, out.data_ptr() + skip * out.element_size(),
                           native.FP16 if out_half else native.FP32, pitch, stream)
        self.torch.cuda.synchronize()
        flat = out.cpu().numpy()
        assert (flat[:skip] == 55).all()
        full = flat[skip:].reshape(rows, pitch)
        assert (full[:, classes:] == 55).all()
        return full[:, :classes]

    def check_ruled(self, **kw):
        got = self.ruled(**kw)
        lo, hi = self.line_at[0], self.line_at[-1]
        with np.errstate(over="ignore"):
            want = self.want.astype(got.dtype)
        assert np.array_equal(got[lo:hi], want[lo:hi], equal_nan=True)
        assert (got[:lo] == 55).all() and (got[hi:] == 55).all()

    def buffers(self):
        t, (rows, lines) = self.torch, (len(self.z), len(self.line_at) - 1)
        whole = dict(dtype=t.int32, device="cuda")
        return [t.full((lines,), 9, **whole), t.full((rows,), 9, **whole), t.full((rows,), 9, **whole),
                t.full((rows,), 9.0, device="cuda")]

    def greedy(self, stream=0, into=None):
        b = into or self.buffers()
        native.ctc_greedy_lines(self.frames, self.crules, *[x.data_ptr() for x in b], stream=stream)
        return b

    def check_greedy(self, got=None):
        got = got or self.greedy()
        self.torch.cuda.synchronize()
        counts, ids, starts, probs = (x.cpu().numpy() for x in got)
        at = self.line_at
        tol = R.sum_tolerance(self.z.shape[1])
        for i, (wid, wst, wpr) in enumerate(R.greedy(self.want, at)):
            n, a, e = len(wid), at[i], at[i + 1]
            assert counts[i] == n, i
            assert ids[a:a + n].tolist() == wid and starts[a:a + n].tolist() == wst, i
            assert np.all(np.abs(probs[a:a + n] - wpr) <= tol * np.array(wpr) + 1e-37), i
            assert (ids[a + n:e] == -1).all() and (starts[a + n:e] == -1).all() and (probs[a + n:e] == 0).all()
        for x in (ids, starts, probs):
            assert (x[:at[0]] == 9).all() and (x[at[-1]:] == 9).all()

    def candidates(self, k, stream=0):
        t, rows = self.torch, len(self.z)
        out = [t.full((rows, max(k, 1)), 9, dtype=t.int32, device="cuda"), t.full((rows, max(k, 1)), 9.0, device="cuda"),
               t.full((rows,), 9.0, device="cuda")]
        if stream:
            t.cuda.synchronize()  # the fills above ran on another stream
        native.candidates_lines(self.frames, self.crules, k, *[x.data_ptr() for x in out], stream=stream)
        return out

    def check_candidates(self, k, got=None):
        got = got or self.candidates(k)
        self.torch.cuda.synchronize()
        ids, logp, blank = (x.cpu().numpy() for x in got)
        lo, hi = self.line_at[0], self.line_at[-1]
        wid, wlp, wbl = R.candidates(self.want[lo:hi], k)
        # (z - best) rounds once, ln sum within the sum's error and two roundings, the difference once
        tol = R.sum_tolerance(self.z.shape[1])

        def near(a, b):
            with np.errstate(over="ignore"):  # what float32 cannot hold is an infinity
                b = np.where(np.isinf(b.astype(np.float32)), b.astype(np.float32), b)
            fin = np.isfinite(b)
            # the sizes in play: z - best at most |logp| + ln C, ln sum at most ln C, the result itself
            room = tol + 2.0 ** -24 * (2 * np.abs(b[fin]) + 4 * np.log(self.z.shape[1] + 1) + 1)
            return np.array_equal(a[~fin], b[~fin].astype(np.float32)) and np.all(np.abs(a[fin] - b[fin]) <= room)

        if k:
            assert np.array_equal(ids[lo:hi], wid)
            assert near(logp[lo:hi], wlp)
            assert (ids[:lo] == 9).all() and (ids[hi:] == 9).all() and (logp[hi:] == 9).all()
        assert near(blank[lo:hi], wbl)
        assert (blank[:lo] == 9).all() and (blank[hi:] == 9).all()


# lengths of lines from none and one frame to long ones; classes under, at and over what a warp or a block takes
SHAPES = [
    (2, [1], 0, 0), (3, [5, 0, 1], 2, 3), (33, [0, 7, 33, 1, 0], 0, 1), (400, [40, 1, 1, 1, 64], 1, 0),
    (800, [62, 0, 128, 3], 0, 5), (801, [31, 32, 33], 0, 0), (1024, [9, 2], 0, 0), (1025, [4, 11], 0, 2),
    (1500, [40, 1], 0, 0), (4099, [5, 6], 0, 0), (12000, [3, 9, 1], 0, 1), (16385, [4, 1], 0, 0), (40001, [3], 0, 1),
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("classes,lengths,first,tail", SHAPES)
def test_the_three_calls_at_every_size(classes, lengths, first, tail, half):
    rng = np.random.default_rng(classes + half)
    at = line_places(rng, lengths, first)
    z = logits_of(rng, at[-1] + tail, classes, half)
    c = Case(z, at, some_rules(rng, len(lengths), classes))
    c.check_ruled()
    c.check_ruled(out_half=True)
    c.check_greedy()
    for k in {0, 1, min(10, classes - 1), min(16, classes - 1)}:
        c.check_candidates(k)


@pytest.mark.parametrize("parts", [(), ("history",), ("bias",), ("allowed",), ("history", "allowed")])
def test_each_rule_alone(parts):
    rng = np.random.default_rng(5 + len(parts))
    lengths = [17, 1, 0, 40, 2]
    at = line_places(rng, lengths)
    c = Case(logits_of(rng, at[-1], 800, False), at, some_rules(rng, 5, 800, parts=parts))
    c.check_ruled()
    c.check_greedy()
    c.check_candidates(12)


def test_parts_left_out_within_the_rules():
    """Penalties, table indexes and set indexes that are null: repeat 1, no penalty, table 0, set 0."""
    rng = np.random.default_rng(8)
    at = line_places(rng, [6, 9, 1])
    z = logits_of(rng, at[-1], 500, False)
    full = some_rules(rng, 3, 500)
    for gone in (("repeat",), ("presence", "frequency"), ("bias_of",), ("set_of",), ("repeat", "presence", "bias_of", "set_of")):
        rules = {k: v for k, v in full.items() if k not in gone}
        c = Case(z, at, rules)
        c.check_ruled()
        c.check_greedy()
        c.check_candidates(5)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("pitch,skip", [(803, 0), (808, 1), (1000, 8), (832, 2)])
def test_strides_and_alignments(pitch, skip, half):
    rng = np.random.default_rng(pitch)
    at = line_places(rng, [21, 1, 13])
    c = Case(logits_of(rng, at[-1] + 2, 800, half), at, some_rules(rng, 3, 800), pitch, skip)
    c.check_ruled(pitch=pitch, skip=skip)
    c.check_ruled(out_half=True, pitch=801, skip=3)
    c.check_greedy()
    c.check_candidates(16)


@pytest.mark.parametrize("classes", [7, 800, 12000])
def test_ties_take_the_lowest_class(classes):
    rng = np.random.default_rng(classes)
    at = line_places(rng, [30, 11, 8])
    z = logits_of(rng, at[-1], classes, True, grid=True)
    z[3] = 1.5  # every class alike
    z[4] = -np.inf
    z[5, 1:] = -np.inf
    c = Case(z, at, None)
    c.check_ruled()
    c.check_greedy()
    c.check_candidates(min(16, classes - 1))
    c = Case(z, at, some_rules(rng, 3, classes, parts=("allowed",)))
    c.check_greedy()
    c.check_candidates(min(16, classes - 1))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("classes", [64, 800, 12000])
def test_nan_and_infinities_where_the_rules_forbid(classes, half):
    """What a forbidden class holds never shows: NaN, infinities, the type's lowest and highest value."""
    rng = np.random.default_rng(classes + 1)
    at = line_places(rng, [20, 20, 6])
    z = logits_of(rng, at[-1], classes, half)
    bad = rng.random(classes) < 0.3
    bad[0] = bad[3] = False
    lim = np.finfo(z.dtype)
    z[:, bad] = rng.choice(np.array([np.nan, np.inf, -np.inf, lim.min, lim.max], z.dtype), (len(z), bad.sum()))
    words = (classes + 31) // 32
    keep = np.zeros(words * 32, bool)
    keep[:classes] = ~bad
    rules = some_rules(rng, 3, classes, parts=("history",))
    rules["allowed"] = (keep.reshape(1, words, 32) * (1 << np.arange(32, dtype=np.uint64))).sum(2).astype(np.uint32)
    c = Case(z, at, rules)
    assert np.isfinite(c.want[:, ~bad]).all()
    c.check_ruled()
    c.check_greedy()
    c.check_candidates(16)
    # the same by a bias of -inf
    rules.pop("allowed")
    rules["bias"] = np.where(bad, -np.inf, 0.25).astype(np.float32)[None]
    c = Case(z, at, rules)
    c.check_ruled()
    c.check_greedy()
    c.check_candidates(16)


def test_a_nan_that_is_allowed_wins_nothing_and_shows():
    rng = np.random.default_rng(2)
    z = logits_of(rng, 6, 100, False)
    z[:, 0] = -20
    z[2, 50] = np.nan
    c = Case(z, np.array([0, 6], np.int32), None)
    out = c.ruled()
    assert np.isnan(out[2, 50]) and np.isnan(out).sum() == 1
    ids, logp, blank = (x.cpu().numpy() for x in c.candidates(4))
    assert np.isnan(blank[2]) and np.isnan(logp[2]).all() and (ids[2] != 50).all()
    assert np.isfinite(np.delete(logp, 2, 0)).all()


def test_lines_of_one_frame():
    """A beam's rows: every row a line with its own history."""
    rng = np.random.default_rng(77)
    for classes in (800, 12000):
        at = np.arange(131, dtype=np.int32)
        c = Case(logits_of(rng, 130, classes, classes > 1000), at, some_rules(rng, 130, classes, longest=200))
        c.check_ruled()
        c.check_greedy()
        c.check_candidates(7)


def test_many_short_and_empty_lines():
    """Thousands of lines: their search, and lengths of none between them."""
    rng = np.random.default_rng(6)
    lengths = rng.integers(0, 4, 3000)
    lengths[:40] = 0
    lengths[-40:] = 0
    at = line_places(rng, lengths)
    c = Case(logits_of(rng, at[-1] + 4, 37, False), at, some_rules(rng, 3000, 37, longest=6))
    c.check_ruled()
    c.check_greedy()
    c.check_candidates(3)


@pytest.mark.parametrize("length", [31, 32, 33, 1000])
def test_a_character_over_many_frames(length):
    """One character held over the collapse's steps, its probability the highest of all its frames."""
    rng = np.random.default_rng(length)
    z = rng.normal(0, 1, (length + 3, 50)).astype(np.float32)
    z[:, 7] += 12
    z[length // 2, 7] += 5
    z[length, 7] = -5  # a break, then the same again
    c = Case(z, np.array([0, length + 3], np.int32), None)
    c.check_greedy()


def test_history_of_a_long_line():
    """Counts past 16 bits."""
    rng = np.random.default_rng(12)
    rules = {"history": np.concatenate([np.full(70001, 5), np.arange(64)]).astype(np.int32),
             "history_at": np.array([0, 70065], np.int32), "frequency": np.array([0.001], np.float32)}
    c = Case(logits_of(rng, 5, 64, False), np.array([0, 5], np.int32), rules)
    c.check_ruled()
    c.check_greedy()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("classes", [300, 800, 2000, 12000])
def test_a_history_that_names_every_class(classes, half):
    """More distinct characters than any list of them keeps, in some lines and not in others."""
    rng = np.random.default_rng(classes)
    lengths = [9, 2, 1, 12]
    at = line_places(rng, lengths)
    ids = [rng.permutation(classes), rng.integers(0, classes, 50), np.concatenate([np.arange(classes), np.arange(0, classes, 3)]),
           rng.integers(0, classes, 5)]
    rules = some_rules(rng, 4, classes)
    rules["history"] = np.concatenate(ids).astype(np.int32)
    rules["history_at"] = np.concatenate([[0], np.cumsum([len(i) for i in ids])]).astype(np.int32)
    c = Case(logits_of(rng, at[-1], classes, half), at, rules)
    c.check_ruled()
    c.check_greedy()
    c.check_candidates(16)
    native.logit_rules(c.frames, c.crules, c.frames.logits, c.kind)  # in place
    c.torch.cuda.synchronize()
    with np.errstate(over="ignore"):
        assert np.array_equal(c.keep[0].cpu().numpy().reshape(-1, classes), c.want.astype(c.z.dtype), equal_nan=True)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("classes,pitch", [(1030, 1030), (1500, 1501), (4096, 4096), (12000, 12000), (16384, 16390)])
def test_long_rows_in_long_lines(classes, pitch, half):
    """Rows past what a warp holds at once, many of them a line: ties, histories that fit and that do not,
    NaN where the rules forbid, a line behind the first block's."""
    rng = np.random.default_rng(classes + half)
    lengths = [33, 0, 1, 70, 18, 40]
    at = line_places(rng, lengths, 2)
    z = logits_of(rng, at[-1] + 3, classes, half, grid=classes == 4096)
    rules = some_rules(rng, 6, classes, longest=200)
    h = [rules["history"][rules["history_at"][i]:rules["history_at"][i + 1]] for i in range(6)]
    h[4] = rng.permutation(classes)[:700].astype(np.int32)
    h[5] = np.concatenate([[0, 0, 0], h[5], h[5]]).astype(np.int32)
    rules["history"] = np.concatenate(h)
    rules["history_at"] = np.concatenate([[0], np.cumsum([len(x) for x in h])]).astype(np.int32)
    c = Case(z, at, rules, pitch)
    c.check_greedy()
    for k in (0, 1, 16):
        c.check_candidates(k)
    bad = rng.random(classes) < 0.2
    bad[:4] = False
    z[:, bad] = rng.choice(np.array([np.nan, np.inf], z.dtype), (len(z), bad.sum()))
    z[40, :] = 0.5
    z[41, 1:] = -np.inf
    z[42, 0] = -1200
    rules = {"bias": np.where(bad, -np.inf, 0.0).astype(np.float32)[None]}
    c = Case(z, at, rules, pitch)
    c.check_greedy()
    c.check_candidates(7)
    c = Case(z[:, :classes], at, {"bias": np.where(np.arange(classes) == 0, 0, -np.inf).astype(np.float32)[None]}, pitch)
    c.check_candidates(2)  # nothing but the blank


def test_the_types_lowest_value_everywhere():
    """Rows of the lowest value, as callers mask: a maximum that times log2 e overflows."""
    z = np.full((4, 900), np.finfo(np.float32).min, np.float32)
    z[1, 5] = np.finfo(np.float32).max / 2
    z[2, 700:] = -1
    z[3, 1:] *= np.float32(0.5)
    c = Case(z, np.array([0, 4], np.int32), None)
    c.check_greedy()
    c.check_candidates(3)
    c = Case(np.tile(z, (1, 3)), np.array([0, 4], np.int32), None)
    c.check_greedy()
    c.check_candidates(3)


def test_in_place_and_side_by_side():
    import torch
    rng = np.random.default_rng(3)
    at = line_places(rng, [12, 1, 9])
    c = Case(logits_of(rng, at[-1], 800, False), at, some_rules(rng, 3, 800))
    native.logit_rules(c.frames, c.crules, c.frames.logits, native.FP32)
    torch.cuda.synchronize()
    assert np.array_equal(c.keep[0].cpu().numpy().reshape(-1, 800), c.want)
    c = Case(logits_of(rng, at[-1], 100, False), at, some_rules(rng, 3, 100), pitch=200)
    native.logit_rules(c.frames, c.crules, c.frames.logits + 400, native.FP32, 200)
    torch.cuda.synchronize()
    both = c.keep[0].cpu().numpy().reshape(-1, 200)
    assert np.array_equal(both[:, :100], c.z) and np.array_equal(both[:, 100:], c.want)


def test_streams_graphs_and_two_calls_at_once():
    """Captured on a stream of its own and replayed with new logits, beside a call on another stream."""
    import torch
    rng = np.random.default_rng(9)
    at = line_places(rng, [62, 0, 100, 1])
    a = Case(logits_of(rng, at[-1], 800, False), at, some_rules(rng, 4, 800))
    b = Case(logits_of(rng, at[-1], 800, False), at, some_rules(rng, 4, 800))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    into, other = a.buffers(), b.buffers()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s1):
        a.greedy(stream=torch.cuda.current_stream().cuda_stream, into=into)
    g.replay()
    b.greedy(stream=s2.cuda_stream, into=other)
    cand = b.candidates(9, stream=s1.cuda_stream)
    torch.cuda.synchronize()
    a.check_greedy(into)
    b.check_greedy(other)
    b.check_candidates(9, cand)
    a.z = logits_of(rng, at[-1], 800, False)
    a.keep[0].copy_(torch.from_numpy(a.z.reshape(-1)))
    a.want = R.ruled(a.z, at, a.rules)
    for x in into:
        x.fill_(9)
    g.replay()
    a.check_greedy(into)


def test_the_same_bits_every_time():
    import torch
    rng = np.random.default_rng(10)
    at = line_places(rng, [300, 1, 40])
    c = Case(logits_of(rng, at[-1], 12000, True), at, some_rules(rng, 3, 12000, longest=300))
    first = [x.clone() for x in c.greedy() + c.candidates(16)]
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, c.greedy() + c.candidates(16)))


def test_agrees_with_the_decoder_without_rules():
    """Without rules, the ids and starts of crec_ctc_greedy on the same frames laid out class by class."""
    import torch
    rng = np.random.default_rng(11)
    n, frames, classes = 5, 131, 800
    z = (rng.integers(-24, 25, (n, classes, frames)) * 0.5).astype(np.float32)
    z[:, 0, ::3] += 30
    c = Case(np.ascontiguousarray(z.transpose(0, 2, 1)).reshape(n * frames, classes),
             (np.arange(n + 1) * frames).astype(np.int32), None)
    counts, ids, starts, probs = (x.cpu().numpy() for x in c.greedy())
    d = torch.from_numpy(z).cuda()
    want, _ = native.ctc_greedy(d.data_ptr(), n, classes, frames, [frames] * n)
    for i, w in enumerate(want):
        a, k = i * frames, counts[i]
        assert np.array_equal(ids[a:a + k], w.ids) and np.array_equal(starts[a:a + k], w.frames)
        # crec_ctc_greedy's own sum: 800 adds in class order and exp_neg's error beside ours
        assert np.allclose(probs[a:a + k], w.probs, rtol=R.sum_tolerance(classes) + 808 * 2.0 ** -24, atol=0)


def test_long_offsets():
    """Rows whose offsets pass 32 bits: 270,000 rows of 16,000 places (float16), lines far into them."""
    import torch
    rng = np.random.default_rng(13)
    rows, pitch, classes = 270000, 16000, 40
    far = rows - 9
    big = torch.zeros(rows, pitch, dtype=torch.float16, device="cuda")
    z = logits_of(rng, 9, classes, True)
    big[far:, :classes] = torch.from_numpy(z).cuda()
    at = np.array([far, far + 4, far + 9], np.int32)
    d_at = dev(at)
    frames = native.LineLogits(big.data_ptr(), native.FP16, classes, pitch, rows, 2, d_at.data_ptr())
    blank = torch.zeros(rows, device="cuda")
    ids = torch.zeros(rows, 3, dtype=torch.int32, device="cuda")
    logp = torch.zeros(rows, 3, device="cuda")
    native.candidates_lines(frames, None, 3, ids.data_ptr(), logp.data_ptr(), blank.data_ptr())
    rules = {"bias": rng.normal(0, 1, (1, classes)).astype(np.float32)}
    d_bias = dev(rules["bias"])
    native.logit_rules(frames, native.Rules(bias=d_bias.data_ptr(), biases=1), big.data_ptr() + 2 * 8000, native.FP16, pitch)
    torch.cuda.synchronize()
    assert np.array_equal(ids[far:].cpu().numpy(), R.candidates(z.astype(np.float32), 3)[0])
    want = R.ruled(z, np.array([0, 4, 9]), rules).astype(np.float16)
    assert np.array_equal(big[far:, 8000:8000 + classes].cpu().numpy(), want)
    assert int((big[:far] != 0).sum()) == 0
