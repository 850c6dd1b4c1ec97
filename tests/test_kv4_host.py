"""The 4-bit K/V cache without a GPU: refusals of the C entries and of the Python calls, the
record layout, and the formulas that the GPU tests compare with."""
import types

import pytest
import torch

from fastforward_b200 import _lib as L
from fastforward_b200 import ops
from tests import _kv4 as ref

P = 16  # a non-NULL, 16-byte aligned pointer that no refused call touches


def write(**k):
    a = dict(qkv=P, row_stride=768, qn=P, kn=P, eps=1e-6, cos=P, sin=P, yq=P, pages=P, num=4, table=P, stride=4,
             width=4, start=P, ctx=P, B=1, T=3, HQ=4, HK=1) | k
    L.call("ffb_qk_norm_rope_kv4", *a.values(), None)


def attend(**k):
    a = dict(q=P, pages=P, num=4, table=P, stride=4, width=4, start=P, ctx=P, out=P, ws=P, bytes=1 << 40, B=1, T=3,
             most=1, HQ=4, HK=1, scale=0.1, window=0, sinks=0) | k
    L.call("ffb_attention_kv4", *a.values(), None)


def read(**k):
    a = dict(pages=P, num=4, table=P, stride=4, width=4, start=P, ctx=P, k=P, v=P, B=1, T=3, HK=1) | k
    L.call("ffb_kv4_read", *a.values(), None)


@pytest.mark.parametrize("f", [write, attend, read])
@pytest.mark.parametrize("bad,match", [
    (dict(pages=None), "NULL"), (dict(table=None), "NULL"), (dict(start=None), "NULL"), (dict(ctx=None), "NULL"),
    (dict(pages=8), "aligned"), (dict(table=18), "alignment"), (dict(num=0), "bad shape"), (dict(width=0), "bad shape"),
    (dict(B=0), "bad shape"), (dict(T=0), "bad shape"), (dict(HK=0), "bad shape"), (dict(T=-1), "bad shape"),
    (dict(B=2, stride=3), "stride"), (dict(width=(1 << 24) + 1, stride=1 << 25), "table width"), (dict(B=70000), "too large")])
def test_common_refusals(f, bad, match):
    with pytest.raises(ValueError, match=match):
        f(**bad)


@pytest.mark.parametrize("bad,match", [
    (dict(qkv=None), "NULL"), (dict(yq=None), "NULL"), (dict(HQ=3, HK=2), "heads"), (dict(row_stride=764), "row_stride"),
    (dict(row_stride=770), "row_stride"), (dict(qkv=20), "aligned"), (dict(cos=4), "aligned"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps")])
def test_write_refusals(bad, match):
    with pytest.raises(ValueError, match=match):
        write(**bad)


@pytest.mark.parametrize("bad,match", [
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(q=8), "aligned"), (dict(out=24), "aligned"),
    (dict(HQ=5, HK=2), "heads"), (dict(most=0), "max_rows"), (dict(most=4), "max_rows"), (dict(scale=float("inf")), "scale"),
    (dict(window=-1), "window"), (dict(sinks=-1, window=2), "sinks"), (dict(sinks=4), "sinks"),
    (dict(window=(1 << 30) + 1), "window"), (dict(T=1 << 24, HQ=128, HK=1), "too large"),
    (dict(width=4096, stride=4096, bytes=64), "workspace"), (dict(width=4096, stride=4096, ws=None), "workspace")])
def test_attention_refusals(bad, match):
    with pytest.raises(ValueError, match=match):
        attend(**bad)


def test_read_refusals():
    for bad, match in ((dict(k=None), "NULL"), (dict(v=40), "aligned")):
        with pytest.raises(ValueError, match=match):
            read(**bad)


def test_workspace_is_zero_for_bad_shapes_and_bounded():
    f = L.lib().ffb_attention_kv4_workspace
    assert f(0, 1, 4, 1, 1, 1, 0, 0) == 0 and f(1, 1, 3, 2, 1, 1, 0, 0) == 0
    assert f(1, 1, 32, 8, 1, 1, 0, 0) == 0  # one page is not shared out
    many = f(1, 1, 32, 8, 1, 4096, 0, 0)
    assert 0 < many <= 8 << 20 and many == f(1, 1, 32, 8, 1, 1 << 24, 0, 0)  # the context's length does not count
    assert f(1, 1, 32, 8, 1, 4096, 64, 0) == 0  # a window bounds the pages
    assert 0 < f(1, 64, 32, 8, 64, 4096, 0, 0) <= 64 * 64 * 32 * 130 * 4


def test_python_calls_refuse_cpu_tensors():
    pages = torch.zeros(1, 1, L.KV4_RECORD, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    n = types.SimpleNamespace(weight=torch.ones(128, dtype=torch.bfloat16), variance_epsilon=1e-6)
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qk_pair_kv4(torch.zeros(1, 384, dtype=torch.bfloat16), n, n, x, x, pages, i[:1, None], i, i[:1])
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_kv4(torch.zeros(1, 1, 128, dtype=torch.bfloat16), pages, i[:1, None], i, i[:1], 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_read(pages, i[:1, None], i, i[:1], 1)
    with pytest.raises(ValueError, match="positive"):
        ops.kv4_pages(0, 1, device="cpu")
    assert ops.kv4_pages(2, 3, device="cpu").shape == (2, 3, L.KV4_RECORD)


def test_layout_round_trip():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 2, 64, 128, generator=g, dtype=torch.float64) for _ in range(2))
    pages = ref.pack(k, v)
    assert pages.shape[-1] == L.KV4_RECORD
    for x, y in zip((k, v), ref.unpack(pages)):
        assert torch.equal(y, ref.values(*ref.quantize(x)))
        assert torch.equal(y, y.to(torch.bfloat16).double())  # every held value is exact in bf16
        step = ref.quantize(x)[1].repeat_interleave(32, -1)
        assert ((x - y).abs() <= step / 2).all()


def test_scales_have_five_significant_bits():
    x = torch.rand(1000, dtype=torch.float64) * 10 + 1e-9
    s = ref.up5(x)
    m, _ = torch.frexp(s)
    assert torch.equal(m * 32, torch.round(m * 32)) and (s >= x).all() and (s <= x * (1 + 1 / 16)).all()


def test_formula_of_attention_is_a_softmax():
    """The tests' formula against torch's own softmax on dense tensors, and its empty rows."""
    g = torch.Generator().manual_seed(2)
    pages = ref.pack(*(torch.randn(3, 2, 64, 128, generator=g, dtype=torch.float64) for _ in range(2)))
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    q = torch.randn(4, 5, 128, generator=g).to(torch.bfloat16)
    starts, lens = torch.tensor([0, 5], dtype=torch.int32), torch.tensor([100], dtype=torch.int32)
    got, _ = ref.attention(q, pages, table, starts, lens, 0.1, 0, 0)
    k, v = (x[[2, 0]].transpose(0, 1).reshape(2, 128, 128)[:, :100].repeat_interleave(2, 0) for x in ref.unpack(pages))
    mask = torch.arange(100)[None] <= torch.arange(95, 100)[:, None]
    want = torch.softmax((q.double() @ k.transpose(1, 2) * 0.1).masked_fill(~mask, -torch.inf), -1) @ v
    assert torch.allclose(got, want.transpose(0, 1), atol=1e-12)
    got, _ = ref.attention(q, pages, table, starts, torch.tensor([2], dtype=torch.int32), 0.1, 0, 0)
    assert not got[:3].any() and got[3:].any()
