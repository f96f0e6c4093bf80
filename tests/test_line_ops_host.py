"""What the calls on packed lines' logits and the head with adapters refuse, before any GPU call."""
from __future__ import annotations

import struct

import numpy as np
import pytest

from carbon_rec import native

Z = dict(logits=64, type=native.FP32, classes=10, pitch=10, rows=4, lines=2, line_at=64)


def frames(**kw):
    return native.LineLogits(**{**Z, **kw})


def refused(code, call, *args, **kw):
    with pytest.raises(native.CrecError) as e:
        call(*args, **kw)
    assert e.value.code == code and str(e.value)
    return str(e.value)


CALLS = [lambda z, r=None: native.logit_rules(z, r, 4096), lambda z, r=None: native.ctc_greedy_lines(z, r, 64, 64, 64, 64),
         lambda z, r=None: native.candidates_lines(z, r, 3, 64, 64, 64)]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("wrong", [dict(type=0), dict(type=7), dict(classes=0), dict(classes=-3), dict(pitch=9), dict(pitch=1 << 41),
                                   dict(rows=-1), dict(rows=1 << 31), dict(lines=-1), dict(line_at=0), dict(logits=0),
                                   dict(logits=66), dict(logits=65, type=native.FP16), dict(line_at=66),
                                   dict(pitch=1 << 40, rows=1 << 30), dict(rows=(1 << 31) - 255)])
def test_logits_that_are_refused(call, wrong):
    refused(native.E_INVALID, call, frames(**wrong))


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("wrong", [dict(history=64), dict(history_at=64), dict(repeat=64), dict(presence=64), dict(bias=64),
                                   dict(bias_of=64), dict(bias=64, biases=-1), dict(allowed=64), dict(set_of=64),
                                   dict(allowed=64, sets=0), dict(history=66, history_at=64), dict(bias=65, biases=1),
                                   dict(allowed=64, sets=1, set_of=62)])
def test_rules_that_are_refused(call, wrong):
    refused(native.E_INVALID, call, frames(), native.Rules(**wrong))


@pytest.mark.parametrize("out,kind,pitch", [(0, native.FP32, 10), (4098, native.FP32, 10), (4097, native.FP16, 10),
                                            (4096, 0, 10), (4096, native.FP32, 9), (68, native.FP32, 10), (64, native.FP16, 10),
                                            (64, native.FP32, 12), (104, native.FP32, 10), (32, native.FP32, 10)])
def test_outputs_of_the_rules_that_are_refused(out, kind, pitch):
    refused(native.E_INVALID, native.logit_rules, frames(), None, out, kind, pitch)


def test_outputs_beside_the_logits():
    """In rows of the same byte pitch: beside them passes (no GPU here: the next check fails), on them does not."""
    import torch
    wide = frames(pitch=20)
    for at in (64 + 36, 64 - 36, 64 + 44, 64 - 44):
        assert "overlaps" in refused(native.E_INVALID, native.logit_rules, wide, None, at, native.FP32, 20)
    if not torch.cuda.is_available():
        for at in (64 + 40, 64 + 40 - 80, 64 + 40 + 80):
            refused(native.E_CUDA, native.logit_rules, wide, None, at, native.FP32, 20)


@pytest.mark.parametrize("k", [-1, 10, 17, 100])
def test_topk_out_of_range(k):
    refused(native.E_RANGE, native.candidates_lines, frames(), None, k, 64, 64, 64)
    refused(native.E_RANGE, native.candidates_lines, frames(classes=100, pitch=100), None, max(k, 17), 64, 64, 64)


def test_outputs_that_are_missing():
    for i in range(4):
        out = [0 if j == i else 64 for j in range(4)]
        refused(native.E_INVALID, native.ctc_greedy_lines, frames(), None, *out)
    refused(native.E_INVALID, native.ctc_greedy_lines, frames(), None, 64, 64, 66, 64)
    refused(native.E_INVALID, native.candidates_lines, frames(), None, 3, 64, 65, 64)
    for out in ((0, 64, 64), (64, 0, 64), (64, 64, 0)):
        refused(native.E_INVALID, native.candidates_lines, frames(), None, 3, *out)


def test_nothing_to_do():
    for z in (frames(lines=0, line_at=0), frames(lines=0, rows=0, logits=0)):
        for call in CALLS:
            call(z)
    native.logit_rules(frames(rows=0, logits=0), None, 0)
    native.candidates_lines(frames(rows=0, logits=0), None, 3, 0, 0, 0)


def head(k=16, classes=5):
    w, b = np.zeros((classes, k), np.float16), np.zeros(classes, np.float32)
    return native.ctc_head_blob(b"CTCHEAD1" + struct.pack("<ii", classes, k) + w.tobytes() + b.tobytes())


def adapter(k=16, classes=5, rank=2):
    return np.zeros((rank, k), np.float16), np.zeros((classes, rank), np.float16), 1.0


def test_blob_head(rec_latin):
    assert native.blob_head(head(24, 7)) == (24, 7)
    assert native.blob_head(rec_latin[1].to_blob()) == (256, 800)


def test_blobs_that_are_refused(rec_latin):
    good = head()
    bad = [b"", b"CRECMDL1", good[:-1], good + b"\0", b"X" + good[1:], good[:60], rec_latin[0].to_blob()]
    for at, v in ((8, 2), (12, 0), (16, 5000), (20, 0), (20, 9), (88, 2), (88 + 16, 3), (88 + 24, 2), (88 + 32, 1), (88 + 48, 0),
                  (88 + 48, 1 << 30), (88 + 52, 0x7fffffff), (88 + 56, 1), (88 + 76, 1)):
        bad.append(good[:at] + struct.pack("<I", v) + good[at + 4:])
    for blob in bad:
        refused(native.E_MODEL, native.blob_head, blob)
        refused(native.E_MODEL, native.Adapters, blob)


def test_adapters_that_are_refused():
    for k, classes, sets, code in ((12, 5, [], native.E_MODEL), (520, 5, [], native.E_MODEL),
                                   (16, 5, [adapter(rank=65)], native.E_RANGE), (16, 5, [adapter(rank=0)], native.E_RANGE),
                                   (16, 5, [adapter(k=24)], native.E_INVALID), (16, 5, [adapter(classes=6)], native.E_INVALID)):
        refused(code, native.Adapters, head(k, classes), sets)
    a, b, s = adapter()
    refused(native.E_INVALID, native.Adapters, head(), [(a, b.T, s)])
    refused(native.E_INVALID, native.Adapters, head(), [adapter()], device=-1)


def test_closing_nothing():
    assert native.lib().crec_adapters_close(None) == native.OK
