"""More lines than the calls on packed lines' logits count in 32 bits: refused, before any GPU call."""
from __future__ import annotations

import pytest

from carbon_rec import native
from test_line_ops_host import CALLS, frames, refused


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("lines", [(1 << 31) - 1, (1 << 31) - 255])
def test_more_lines_than_there_may_be(call, lines):
    assert "lines" in refused(native.E_INVALID, call, frames(lines=lines))
