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


def _attend(**k):
    a = dict(q=P, pages=P, num=4, table=P, stride=4, width=4, start=P, ctx=P, out=P + (1 << 20), ws=P, bytes=1 << 40, B=1, T=3,
             most=1, HQ=4, HK=1, scale=0.1, window=0, sinks=0) | k
    L.call("ffb_attention_kv4", *a.values(), None)


@pytest.mark.parametrize("scale", [3e38, -2.5e38, float("inf"), float("nan")])
def test_scales_that_overflow_in_base_2_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        _attend(scale=scale)


def _write(**k):
    a = dict(qkv=P, row_stride=768, qn=P, kn=P, eps=1e-6, cos=P, sin=P, yq=P + (1 << 20), pages=P, num=4, table=P, stride=4,
             width=4, start=P, ctx=P, B=1, T=3, HQ=4, HK=1) | k
    L.call("ffb_qk_norm_rope_kv4", *a.values(), None)


@pytest.mark.parametrize("f,bad", [
    (_attend, dict(out=P)), (_attend, dict(out=P + 3 * 4 * 256 - 16)), (_attend, dict(out=P - 3 * 4 * 256 + 16)),
    (_attend, dict(T=1, out=P + 16)), (_attend, dict(HQ=1, out=P + 16)), (_write, dict(yq=P)), (_write, dict(yq=P + 256)),
    (_write, dict(T=1, yq=P + 8)), (_write, dict(yq=P + (2 * 768 + 6 * 128) * 2 - 8)), (_write, dict(yq=P - 3 * 4 * 256 + 8))])
def test_overlapping_results_are_refused(f, bad):
    """A CTA stores its rows while others have yet to read theirs."""
    with pytest.raises(ValueError, match="overlap"):
        f(**bad)


@pytest.mark.parametrize("at,value", [(0, 65536), (1, 1 << 25), (1, 1 << 30), (2, 4104), (3, 1 << 30), (4, 65), (5, (1 << 24) + 1),
                                      (6, (1 << 30) + 1), (7, (1 << 30) + 1)])
def test_workspace_of_refused_shapes_is_zero(at, value):
    f = L.lib().ffb_attention_kv4_workspace
    shape = [2, 64, 32, 8, 64, 4096, 1 << 20, 4]
    assert f(*shape) > 0
    shape[at] = value
    if at == 3:
        shape[2] = value
    assert f(*shape) == 0
