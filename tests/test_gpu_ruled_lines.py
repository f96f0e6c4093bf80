"""Lines recognised by a device, decoded again under adapters and rules: the head's input of the last run
(crec_head_input), the head with adapters (crec_adapters_logits), the rules (crec_logit_rules), greedy
CTC and the beam's candidates under them (crec_ctc_greedy_lines, crec_candidates_lines), as they are
used together."""
from __future__ import annotations

import numpy as np
import pytest

import line_ref as R
from carbon_rec import native, synth

pytestmark = pytest.mark.gpu

FP16_HEAD_TOL = 2 * (256 + 2) * 2.0 ** -23  # two float32 sums of 256 products and a bias, of their magnitudes


def recognised(rec_latin, precision):
    pages, boxes = synth.pages(31, 2, 1600, 1200, 12)
    page_of = np.repeat(np.arange(2), 12).astype(np.int32)
    blob = rec_latin[0 if precision == native.INT8 else 1].to_blob()
    dev = native.RecDevice(blob, precision, max_lines=32, max_width=1024, max_pages=2)
    dev.set_pages(pages)
    dev.arm_logits()
    lines, lengths = dev.recognize(page_of, np.concatenate(boxes), 1024)
    return dev, lines, lengths, dev.logits([1024] * 24, 800)


def features(dev, rows, lengths):
    import torch
    total = int(sum(lengths[r] for r in rows))
    x = torch.full((total + 5, 256), 9.0, dtype=torch.float16, device="cuda")
    at = dev.head_input(rows, x.data_ptr(), 256, total)
    assert at.tolist() == np.concatenate([[0], np.cumsum([lengths[r] for r in rows])]).tolist()
    assert (x[total:] == 9).all()
    return x, at


def test_head_input_int8(rec_latin):
    """The codes' values of the head's input value, frame by frame."""
    dev, _, lengths, _ = recognised(rec_latin, native.INT8)
    try:
        net = rec_latin[0]
        v = net.layers[-1].inp
        q = dev.value(v, 24 * 256 * 256).reshape(24, 256, 256)
        rows = [3, 0, 17, 23, 3]
        x, at = features(dev, rows, lengths)
        x = x.cpu().numpy()
        for j, r in enumerate(rows):
            want = ((q[r, :lengths[r]].astype(np.int32) - net.values[v].zero).astype(np.float32) *
                    np.float32(net.values[v].scale)).astype(np.float16)
            assert np.array_equal(x[at[j]:at[j + 1]], want)
        for bad, code in ((lambda: dev.head_input([24], 64, 256, 999), native.E_RANGE),
                          (lambda: dev.head_input([0], 64, 255, 999), native.E_INVALID),
                          (lambda: dev.head_input([0, 1], 64, 256, int(lengths[0])), native.E_RANGE),
                          (lambda: dev.head_input([0], 0, 256, 999), native.E_INVALID)):
            with pytest.raises(native.CrecError) as e:
                bad()
            assert e.value.code == code
        assert dev.head_input([], 0, 256, 0).tolist() == [0]
    finally:
        dev.close()


def test_lines_again_under_adapters_and_rules(rec_latin):
    import torch
    dev, lines, lengths, logits = recognised(rec_latin, native.FP16)
    try:
        rows = list(range(24))
        x, at = features(dev, rows, lengths)
        d_at = torch.from_numpy(at).cuda()
        total, n = int(at[-1]), len(rows)
        blob = rec_latin[1].to_blob()
        rng = np.random.default_rng(5)
        sets = [(rng.normal(0, 1 / 16, (r, 256)).astype(np.float16), rng.normal(0, 0.1, (800, r)).astype(np.float16), 1.5)
                for r in (16, 4)]
        head = native.Adapters(blob, sets)
        z = torch.zeros(total, 800, device="cuda")
        # the head alone: the run's own logits but for the sums' order
        head.logits(x.data_ptr(), total, n, d_at.data_ptr(), 0, z.data_ptr())
        torch.cuda.synchronize()
        own = np.concatenate([logits[r][:, :lengths[r]].T for r in rows])
        layer = rec_latin[1].layers[-1]
        w = np.asarray(layer.wf, np.float32).reshape(800, 256).astype(np.float16)
        _, mag = R.adapters(x[:total].cpu().numpy(), w, np.asarray(layer.bias, np.float32), [], at, None)
        assert np.all(np.abs(z.cpu().numpy() - own) <= FP16_HEAD_TOL * mag)
        # without rules: the run's decodings where no frame is a near tie
        b = [torch.zeros(n, dtype=torch.int32, device="cuda")] + [torch.zeros(total, dtype=t, device="cuda")
                                                                 for t in (torch.int32, torch.int32, torch.float32)]
        frames = native.LineLogits(z.data_ptr(), native.FP32, 800, 800, total, n, d_at.data_ptr())
        native.ctc_greedy_lines(frames, None, *[t.data_ptr() for t in b])
        torch.cuda.synchronize()
        counts, ids, starts, _ = (t.cpu().numpy() for t in b)
        top = np.sort(own, axis=1)[:, -2:]
        clear = (top[:, 1] - top[:, 0]) > 2 * FP16_HEAD_TOL * mag.max(1)
        checked = 0
        for j in rows:
            if clear[at[j]:at[j + 1]].all():
                checked += 1
                assert np.array_equal(ids[at[j]:at[j] + counts[j]], lines[j].ids)
                assert np.array_equal(starts[at[j]:at[j] + counts[j]], lines[j].frames)
        assert checked > n // 2
        # each line its adapter and rules: digits and the blank for some, what it read already penalised
        adapter = torch.from_numpy(rng.integers(-1, 2, n).astype(np.int32)).cuda()
        bits = np.zeros((1, 25 * 32), bool)
        bits[0, [0] + list(range(16, 60))] = True
        rules = {"history": np.concatenate([l.ids for l in lines]).astype(np.int32),
                 "history_at": np.concatenate([[0], np.cumsum([len(l.ids) for l in lines])]).astype(np.int32),
                 "repeat": np.full(n, 1.2, np.float32), "frequency": np.full(n, 0.1, np.float32),
                 "bias": rng.normal(0, 0.5, (1, 800)).astype(np.float32),
                 "allowed": (bits.reshape(1, 25, 32) * (1 << np.arange(32, dtype=np.uint64))).sum(2).astype(np.uint32),
                 "set_of": (np.arange(n) % 3 - 1).astype(np.int32)}
        d = {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for k, v in rules.items()}
        c_rules = native.Rules(biases=1, sets=1, **{k: v.data_ptr() for k, v in d.items()})
        ruled = torch.zeros(total, 800, device="cuda")
        cand = [torch.zeros(total, 5, dtype=torch.int32, device="cuda"), torch.zeros(total, 5, device="cuda"),
                torch.zeros(total, device="cuda")]
        head.logits(x.data_ptr(), total, n, d_at.data_ptr(), adapter.data_ptr(), z.data_ptr())
        native.logit_rules(frames, c_rules, ruled.data_ptr())
        native.ctc_greedy_lines(frames, c_rules, *[t.data_ptr() for t in b])
        native.candidates_lines(frames, c_rules, 5, *[t.data_ptr() for t in cand])
        torch.cuda.synchronize()
        want, mag = R.adapters(x[:total].cpu().numpy(), w, np.asarray(layer.bias, np.float32), sets, at, adapter.cpu().numpy())
        got = z.cpu().numpy()
        assert np.all(np.abs(got - want) <= (2 * 256 + 2 * 16 + 8) * 2.0 ** -23 * mag)
        want = R.ruled(got, at, rules)
        assert np.array_equal(ruled.cpu().numpy(), want)
        counts, ids, starts, probs = (t.cpu().numpy() for t in b)
        for j, (wid, wst, wpr) in enumerate(R.greedy(want, at)):
            a, k = at[j], counts[j]
            assert ids[a:a + k].tolist() == wid and starts[a:a + k].tolist() == wst
            assert np.allclose(probs[a:a + k], wpr, rtol=R.sum_tolerance(800), atol=0)
        wid, _, _ = R.candidates(want, 5)
        assert np.array_equal(cand[0].cpu().numpy(), wid)
        head.close()
    finally:
        dev.close()
