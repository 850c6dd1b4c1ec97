"""Edges of the 4-bit K/V cache's calls without a GPU: arguments that are refused."""
import pytest
import torch

from fastforward_b200 import _lib as L
from fastforward_b200 import ops

P = 1 << 20  # an aligned pointer that no refused call touches


@pytest.mark.parametrize("bad", [dict(window=1 << 32), dict(window=(1 << 32) + 7), dict(window=-1), dict(window=(1 << 30) + 1),
                                 dict(window=5, sinks=1 << 32), dict(window=5, sinks=-(1 << 32)), dict(window=5, sinks=1 << 31)])
def test_windows_that_do_not_fit_are_refused(bad):
    """A C int would hold the low 32 bits of them: 2^32 as no window at all."""
    pages = torch.zeros(1, 1, L.KV4_RECORD, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="window"):
        ops.attention_kv4(torch.zeros(1, 1, 128, dtype=torch.bfloat16), pages, i[:1, None], i, i[:1], 0.1, **bad)


@pytest.mark.parametrize("rows", [-1, (1 << 24) + 1, 1 << 32, (1 << 32) + 1])
def test_reads_of_rows_that_do_not_fit_are_refused(rows):
    pages = torch.zeros(1, 1, L.KV4_RECORD, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows"):
        ops.kv4_read(pages, i[:1, None], i, i[:1], rows)
