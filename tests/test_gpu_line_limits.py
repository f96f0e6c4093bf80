"""The calls on packed lines' logits and the head with adapters at the most rows and lines."""
from __future__ import annotations

import numpy as np
import pytest

from carbon_rec import native
from test_gpu_adapters import LENGTHS
from test_gpu_adapters import Case as Head
from test_gpu_line_rules import dev

pytestmark = pytest.mark.gpu


def test_the_most_rows():
    """Rows near the most that an array may have, of one class, in place; the lines are its last rows."""
    import torch
    rows = (1 << 31) - 300
    far = rows - 9
    big = torch.zeros(rows, dtype=torch.float16, device="cuda")
    z = np.linspace(-3, 3, 9).astype(np.float16)
    big[far:] = torch.from_numpy(z).cuda()
    d_at, d_bias = dev(np.array([far, far + 4, far + 9], np.int32)), dev(np.array([0.5], np.float32))
    frames = native.LineLogits(big.data_ptr(), native.FP16, 1, 1, rows, 2, d_at.data_ptr())
    native.logit_rules(frames, native.Rules(bias=d_bias.data_ptr(), biases=1), big.data_ptr(), native.FP16)
    torch.cuda.synchronize()
    assert np.array_equal(big[far:].cpu().numpy(), (z.astype(np.float32) + np.float32(0.5)).astype(np.float16))
    assert not bool(big[:far].any())


@pytest.mark.parametrize("lines", [(1 << 31) - 1, (1 << 31) - 255])
def test_more_lines_than_a_head_takes(lines):
    c = Head(64, 40, [8], LENGTHS)
    c.upload()
    h = c.open()
    out = c.queue(h)
    with pytest.raises(native.CrecError) as e:
        h.logits(c.d[0].data_ptr(), c.rows, lines, c.d[1].data_ptr(), c.d[2].data_ptr(), out.data_ptr())
    assert e.value.code == native.E_INVALID and "lines" in str(e.value)
    c.check(out)
    h.close()
