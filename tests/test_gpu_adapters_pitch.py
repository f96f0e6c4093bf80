"""The head with adapters: what lies between the logits' rows, and behind the last, is left as it was."""
from __future__ import annotations

import numpy as np
import pytest

from carbon_rec import native
from test_gpu_adapters import Case

pytestmark = pytest.mark.gpu

# rows of classes that end inside a 16-byte piece, in pitches that are whole pieces: fewer classes than one
# box of 128 bytes, a box and a bit, several chunks, nearly a box
SIZES = [(5, 8), (15, 16), (33, 40), (79, 80), (231, 232), (295, 296), (495, 496), (801, 808), (1359, 1360), (2197, 2200)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lengths,first,tail", [([128, 40, 3], 0, 0), ([1] * 90, 0, 0), ([200, 0, 77], 2, 5)])
@pytest.mark.parametrize("classes,pitch", SIZES)
def test_the_gaps_of_a_pitch(classes, pitch, lengths, first, tail, half):
    c = Case(128, classes, [16, 8], lengths, first, tail)
    c.upload()
    h = c.open()
    c.check(c.queue(h, half, pitch, 8), half, pitch, 8)
    h.close()


@pytest.mark.parametrize("half", [False, True])
def test_an_array_that_ends_with_its_last_class(half):
    """The last row has no gap behind it: another array begins there."""
    import torch
    c = Case(64, 101, [8], [40, 31])
    c.upload()
    kind = torch.float16 if half else torch.float32
    whole = torch.full((c.rows * 104,), 55.0, dtype=kind, device="cuda")
    h = c.open()
    c.queue(h, half, 104, out=whole)
    torch.cuda.synchronize()
    h.close()
    assert (whole.view(c.rows, 104)[:, 101:] == 55).all()
    c.check(whole, half, 104)


def test_two_heads_side_by_side():
    """Two heads' logits in one array, the second's beginning where the first's end."""
    import torch
    a, b = Case(64, 21, [8], [40, 90]), Case(64, 11, [16], [40, 90])
    both = torch.full((a.rows, 32), 55.0, device="cuda")
    for c, at in ((b, 21), (a, 0)):
        c.upload()
        h = c.open()
        h.logits(c.d[0].data_ptr(), c.rows, 2, c.d[1].data_ptr(), c.d[2].data_ptr(), both.data_ptr() + 4 * at, native.FP32, pitch=32)
        torch.cuda.synchronize()
        h.close()
    for c, at in ((a, 0), (b, 21)):
        alone = torch.full((c.rows * c.classes,), 55.0, device="cuda")
        alone.copy_(both[:, at:at + c.classes].reshape(-1))
        c.check(alone)
    assert np.isfinite(both.cpu().numpy()).all()
