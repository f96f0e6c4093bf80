"""The head with low-rank adapters (crec_adapters_logits) against the formula in 64 bits (line_ref.py)."""
from __future__ import annotations

import struct

import numpy as np
import pytest

import line_ref as R
from carbon_rec import native

pytestmark = pytest.mark.gpu


def head_blob(w, b):
    classes, k = w.shape
    return native.ctc_head_blob(b"CTCHEAD1" + struct.pack("<ii", classes, k) + w.tobytes() + b.tobytes())


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Case:
    """A head of k channels to `classes` with adapters of `ranks`, lines of `lengths` frames, each with an
    adapter of which -1 and one past the last are none."""

    def __init__(self, k, classes, ranks, lengths, first=0, tail=0, seed=0, scale=1.0, adapter=True):
        rng = np.random.default_rng(seed + k + classes)
        self.w = rng.normal(0, 0.06, (classes, k)).astype(np.float16)
        self.b = rng.normal(0, 0.5, classes).astype(np.float32)
        self.sets = [((rng.normal(0, scale, (r, k)) / np.sqrt(k)).astype(np.float16),
                      rng.normal(0, 0.1, (classes, r)).astype(np.float16), float(rng.uniform(0.5, 2))) for r in ranks]
        self.line_at = np.concatenate([[first], first + np.cumsum(lengths)]).astype(np.int32)
        self.rows = int(self.line_at[-1]) + tail
        self.x = rng.normal(0, 1, (self.rows, k)).astype(np.float16)
        self.adapter = rng.integers(-1, len(ranks) + 1, len(lengths)).astype(np.int32) if adapter else None
        self.k, self.classes = k, classes

    def open(self):
        return native.Adapters(head_blob(self.w, self.b), self.sets)

    def upload(self, x_pitch=None):
        x_pitch = x_pitch or self.k
        flat = np.full((self.rows, x_pitch), 99, np.float16)
        flat[:, :self.k] = self.x
        self.d = [dev(flat), dev(self.line_at), dev(self.adapter) if self.adapter is not None else None]
        self.x_pitch = x_pitch

    def queue(self, h, half=False, pitch=None, skip=0, stream=0, out=None):
        import torch
        pitch = pitch or self.classes
        if out is None:
            out = torch.full((skip + self.rows * pitch,), 55.0, dtype=torch.float16 if half else torch.float32, device="cuda")
        h.logits(self.d[0].data_ptr(), self.rows, len(self.line_at) - 1, self.d[1].data_ptr(),
                 self.d[2].data_ptr() if self.d[2] is not None else 0, out.data_ptr() + skip * out.element_size(),
                 native.FP16 if half else native.FP32, self.x_pitch, pitch, stream)
        return out

    def check(self, out, half=False, pitch=None, skip=0):
        import torch
        torch.cuda.synchronize()
        pitch = pitch or self.classes
        flat = out.cpu().numpy()
        full = flat[skip:].reshape(self.rows, pitch)
        lo, hi = self.line_at[0], self.line_at[-1]
        assert (flat[:skip] == 55).all() and (full[:, self.classes:] == 55).all()
        assert (full[:lo] == 55).all() and (full[hi:] == 55).all()
        want, mag = R.adapters(self.x, self.w, self.b, self.sets, self.line_at, self.adapter)
        # K products and their adds, the inner sums' K, the rank's adds, the splits and the last adds: each
        # at most one unit 2^-23 (an accumulator that truncates) of the products' magnitudes
        rank = max([a.shape[0] for a, _, _ in self.sets], default=0)
        room = (2 * self.k + 2 * rank + 8) * 2.0 ** -23 * mag
        if half:
            room = room + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
        assert np.all(np.abs(full[lo:hi, :self.classes] - want[lo:hi]) <= room[lo:hi])


LENGTHS = [62, 0, 1, 7, 128, 129, 3]
CASES = [
    (256, 800, [16] * 5, LENGTHS, 0, 0), (256, 800, [8], [1], 0, 0), (192, 1500, [4, 64, 1, 33], LENGTHS, 3, 9),
    (128, 33, [16, 2], [200, 200], 0, 1), (320, 400, [48, 7, 12], LENGTHS, 0, 0), (64, 12000, [32] * 3, [40, 90], 0, 0),
    (8, 2, [1], [5, 130], 0, 0), (512, 801, [64, 64, 5], LENGTHS, 1, 0), (72, 130, [16] * 40, [1] * 300, 0, 5),
    (256, 800, [16] * 30, [8] * 60, 0, 0), (504, 1, [3], [64, 65], 0, 0), (256, 800, [], LENGTHS, 0, 0),
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("k,classes,ranks,lengths,first,tail", CASES)
def test_logits_are_the_formulas(k, classes, ranks, lengths, first, tail, half):
    c = Case(k, classes, ranks, lengths, first, tail)
    c.upload()
    h = c.open()
    c.check(c.queue(h, half), half)
    h.close()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("x_pitch,pitch,skip", [(264, 803, 1), (512, 808, 8), (256, 1000, 2)])
def test_strides_and_alignments(x_pitch, pitch, skip, half):
    c = Case(256, 800, [16, 8, 32], LENGTHS, 2, 5)
    c.upload(x_pitch)
    h = c.open()
    c.check(c.queue(h, half, pitch, skip), half, pitch, skip)


def test_without_line_adapters():
    c = Case(256, 800, [16, 8], LENGTHS, adapter=False)
    c.upload()
    c.check(c.queue(c.open()))


def test_large_inner_sums():
    """Inner sums past float16's range (and its rounding): they are held in float32."""
    c = Case(256, 100, [16, 16], [70, 70, 5], scale=20000.0)
    c.upload()
    inner = c.x[:70].astype(np.float64) @ c.sets[0][0].astype(np.float64).T
    assert np.abs(inner).max() > 65504 / 2
    c.check(c.queue(c.open()))


def test_the_same_adapter_in_lines_apart():
    c = Case(256, 800, [16] * 3, [20, 9, 30, 1, 15, 40, 13], seed=4)
    c.adapter = np.array([2, 0, 2, -1, 0, 2, 1], np.int32)
    c.upload()
    c.check(c.queue(c.open()))


def test_a_run_of_many_lines():
    rng = np.random.default_rng(0)
    c = Case(256, 800, [16] * 12, list(rng.integers(0, 140, 150)), tail=3)
    c.upload()
    h = c.open()
    c.check(c.queue(h))
    c.check(c.queue(h, True), True)


def test_streams_graphs_and_two_calls_at_once():
    import torch
    a = Case(256, 800, [16] * 4, LENGTHS, seed=1)
    b = Case(256, 800, [16] * 4, [90, 1, 300], seed=2)
    a.upload(), b.upload()
    ha, hb = a.open(), b.open()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    out = torch.full((a.rows * 800,), 55.0, device="cuda")
    o2 = [torch.full((b.rows * 800,), 55.0, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s1):
        a.queue(ha, stream=torch.cuda.current_stream().cuda_stream, out=out)
    g.replay()
    for o, s in zip(o2, (s1, s2, s1)):
        b.queue(hb, stream=s.cuda_stream, out=o)
    a.check(out)
    for o in o2:
        b.check(o)
    a.x = np.random.default_rng(3).normal(0, 1, a.x.shape).astype(np.float16)
    a.d[0].copy_(torch.from_numpy(a.x))
    out.fill_(55.0)
    g.replay()
    a.check(out)


def test_a_wait_that_runs_out_ends_the_launch():
    """Nothing loaded: the launch ends, the calls after it say so, and the GPU and other handles go on."""
    import torch
    for lengths in (LENGTHS, [100] * 400):
        c = Case(256, 800, [16, 8], lengths)
        c.upload()
        h = c.open()
        c.check(c.queue(h))
        h.inject()
        c.queue(h)
        torch.cuda.synchronize()
        for call in (lambda: c.queue(h), h.close):
            with pytest.raises(native.CrecError) as e:
                call()
            assert e.value.code == native.E_TIMEOUT
        h = c.open()
        c.check(c.queue(h))
        h.close()


def test_the_same_bits_every_time():
    import torch
    c = Case(192, 1500, [16] * 8, [30] * 40)
    c.upload()
    h = c.open()
    first = c.queue(h).clone()
    for _ in range(3):
        assert torch.equal(first, c.queue(h))
