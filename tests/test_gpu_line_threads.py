"""The calls on packed lines' logits from several threads at once."""
from __future__ import annotations

import threading

import numpy as np
import pytest

from carbon_rec import native
from test_gpu_line_rules import Case, line_places, logits_of, some_rules

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[20] * 30, [1] * 300])
def test_two_threads_with_other_class_counts(lengths):
    """Calls at once from two threads, whose kernels take other amounts of shared memory: none fails, and each
    gets what it gets alone."""
    import torch
    at = line_places(None, lengths)
    cases, alone = [], []
    for classes in (3000, 12000):
        rng = np.random.default_rng(classes)
        c = Case(logits_of(rng, at[-1], classes, True), at, some_rules(rng, len(lengths), classes))
        cases.append(c)
        alone.append([x.clone() for x in c.greedy()] + [x.clone() for x in c.candidates(5)])
    torch.cuda.synchronize()
    faults, ready = [], threading.Barrier(2)
    outs = [[torch.empty_like(x) for x in a] for a in alone]
    streams = [torch.cuda.Stream() for _ in cases]

    def calls(c, out, stream):
        try:
            ready.wait(60)
            for _ in range(1500):
                native.ctc_greedy_lines(c.frames, c.crules, *[x.data_ptr() for x in out[:4]], stream=stream.cuda_stream)
                native.candidates_lines(c.frames, c.crules, 5, *[x.data_ptr() for x in out[4:]], stream=stream.cuda_stream)
        except Exception as e:  # noqa: BLE001 (told by the test)
            faults.append(repr(e))

    threads = [threading.Thread(target=calls, args=a) for a in zip(cases, outs, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not faults
    assert all(torch.equal(x, y) for a, o in zip(alone, outs) for x, y in zip(a, o))
