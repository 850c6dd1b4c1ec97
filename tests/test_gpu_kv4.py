"""The 4-bit K/V cache on the GPU: its writer, its reader and the attention over it, against
plain formulas in 64 bits (tests/_kv4.py)."""
import subprocess
import sys
import types
from pathlib import Path

import pytest
import torch

from fastforward_b200 import _lib as L
from fastforward_b200 import ops
from tests import _kv4 as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(clear=True)
    yield
    assert L.device_error(clear=True) == 0


def _batch(rows, ctx, hk, seed, spare=2, width=None, lead=0, tail=0):
    """Random page table for sequences of ctx tokens whose newest rows are `rows`."""
    g = torch.Generator().manual_seed(seed)
    need = [max(1, -(-c // 64)) for c in ctx]
    num = sum(need) + spare
    order = torch.randperm(num, generator=g).to(torch.int32)
    width = width or max(need)
    table = torch.full((len(ctx), width), -7, dtype=torch.int32)  # unused entries are never read
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([lead] + rows).cumsum(0).to(torch.int32)
    return table, starts, torch.tensor(ctx, dtype=torch.int32), num


def _norm(seed, eps=1e-6):
    g = torch.Generator().manual_seed(seed)
    return types.SimpleNamespace(weight=(1 + 0.2 * torch.randn(128, generator=g)).to(BF16), variance_epsilon=eps)


def _dev(x):
    if isinstance(x, types.SimpleNamespace):
        return types.SimpleNamespace(weight=x.weight.to(DEV), variance_epsilon=x.variance_epsilon)
    return x.to(DEV)


def _written(rows, ctx, hq, hk, seed, lead=0, tail=0, edit=None, weight=None):
    """Runs the writer on random rows; returns everything host-side."""
    table, starts, lens, num = _batch(rows, ctx, hk, seed, lead=lead)
    total = int(starts[-1]) + tail
    g = torch.Generator().manual_seed(seed + 1)
    qkv = torch.randn(total, (hq + 2 * hk) * 128, generator=g).to(BF16)
    if edit:
        edit(qkv)
    angle = torch.rand(total, 128, generator=g) * 6.3
    cos, sin = angle.cos().to(BF16), angle.sin().to(BF16)  # 128 independent columns
    qn, kn = _norm(seed + 2), _norm(seed + 3)
    if weight is not None:
        kn.weight = weight
    pages = ops.kv4_pages(num, hk)
    out = torch.full((hq, total, 128), 7.0, dtype=BF16, device=DEV)
    yq = ops.qk_pair_kv4(_dev(qkv), _dev(qn), _dev(kn), _dev(cos), _dev(sin), pages, _dev(table), _dev(starts),
                         _dev(lens), out=out)
    return types.SimpleNamespace(table=table, starts=starts, lens=lens, qkv=qkv, cos=cos, sin=sin, qn=qn, kn=kn,
                                 pages=pages, yq=yq.cpu(), total=total, hq=hq, hk=hk)


@pytest.mark.parametrize("rows,ctx,hq,hk", [
    ([1], [1], 4, 2), ([1], [64], 8, 8), ([1], [65], 5, 1), ([3, 0, 70], [3, 9, 200], 8, 2), ([130], [131], 16, 4),
    ([1] * 9, [1, 2, 63, 64, 65, 127, 128, 129, 1000], 32, 8), ([600, 0, 113], [611, 5, 500], 6, 3),
    ([700], [700], 5, 1)])
def test_write_and_read_back(rows, ctx, hq, hk):
    c = _written(rows, ctx, hq, hk, seed=11 + len(rows), lead=2, tail=3)
    q, k, v = ref.norm_rotate_quantize(c.qkv, c.qn, c.kn, c.cos, c.sin, hq, hk)
    live = slice(int(c.starts[0]), int(c.starts[-1]))
    gk, gv = (x.cpu() for x in ops.kv4_read(c.pages, _dev(c.table), _dev(c.starts), _dev(c.lens), c.total))
    # keys and values are held exactly as the formula quantises them
    assert torch.equal(gk[:, live].double(), k[:, live])
    assert torch.equal(gv[:, live].double(), v[:, live])
    # the record itself, byte for byte, against the layout's own definition
    want = ref.records(k, v, c)
    held = ref.held_mask(c)
    assert torch.equal(c.pages.cpu()[held], want[held])
    assert int(c.pages.cpu()[~held].count_nonzero()) == 0  # nothing else was written
    # queries: fp32 arithmetic (relative error of a product chain < 8 roundings of 2^-24 on each
    # of the two terms) and one rounding to bf16
    terms = ref.query_terms(c.qkv, c.qn, c.cos, c.sin, hq)
    diff = (c.yq.double() - q)[:, live].abs()
    assert (diff <= q[:, live].abs() * 2.0 ** -8 * 1.01 + terms[:, live] * 2.0 ** -21).all()
    # rows of no sequence are left as they were
    assert (c.yq[:, :live.start] == 7).all() and (c.yq[:, live.stop:] == 7).all()


def test_write_of_special_values():
    """A group with a NaN or an infinity reads as NaN, zeros as zeros, its neighbours as they are."""
    def edit(x):
        x[0, 4 * 128 + 5] = float("nan")           # k head 0: the norm spreads it over the head
        x[1, 5 * 128:6 * 128] = 0                  # v head 0 of row 1: all zero
        x[2, 5 * 128 + 40] = float("inf")          # v head 0 of row 2: group 1 only
        x[3, 5 * 128:5 * 128 + 32] = 2.0 ** -120   # below the smallest held scale
        x[4, 5 * 128:5 * 128 + 32] = 3.0e38
        x[5, 5 * 128:6 * 128] = torch.tensor([7.0, -3.5, 0.5, 1.5] * 32)  # quotients on the border of two codes

    c = _written([6], [6], 4, 1, seed=5, edit=edit)
    gk, gv = (x.cpu() for x in ops.kv4_read(c.pages, _dev(c.table), _dev(c.starts), _dev(c.lens), 6))
    assert gk[0, 0].isnan().all() and not gk[0, 1:].isnan().any()
    assert (gv[0, 1] == 0).all()
    assert gv[0, 2, 32:64].isnan().all() and not gv[0, 2, :32].isnan().any() and not gv[0, 2, 64:].isnan().any()
    assert (gv[0, 3, :32] == 0).all()
    assert gv[0, 4, :32].isnan().all()
    assert gv[0, 5, :4].tolist() == [7.0, -4.0, 0.0, 2.0]  # ties to the even code


@pytest.mark.parametrize("rows", [40, 640])
def test_keys_of_any_size(rows):
    """Rows and norm weights from tiny to huge, rows of zeros: where fp32 leaves its range the keys are
    still the formula's."""
    def edit(x):
        x.mul_(torch.logspace(-30, 25, rows)[:, None])
        x[3] = 0
        x[5, ::3] *= 2.0 ** -40

    weight = _norm(9).weight.float()
    weight[0:40] *= 1e-28
    weight[70:90] *= 1e20
    weight[100:128] *= 1e34
    c = _written([rows], [rows + 3], 4, 1, seed=41, edit=edit, weight=weight.to(BF16))
    x = c.qkv.double().reshape(rows, -1, 128).transpose(0, 1)
    k, v = ref.held(ref.norm_rotate(x[4:5], c.kn, c.cos, c.sin)), ref.held(x[5:])
    gk, gv = (x.cpu().double() for x in ops.kv4_read(c.pages, _dev(c.table), _dev(c.starts), _dev(c.lens), rows))
    assert torch.equal(gk.isnan(), k.isnan()) and torch.equal(gk.nan_to_num(0), k.nan_to_num(0))
    assert torch.equal(gv.isnan(), v.isnan()) and torch.equal(gv.nan_to_num(0), v.nan_to_num(0))


def test_write_strided_rows_and_single_row():
    c = _written([5], [70], 4, 2, seed=21)
    wide = torch.zeros(5, 8 * 128 + 12, dtype=BF16, device=DEV)
    wide[:, 4:4 + 8 * 128] = _dev(c.qkv)
    pages = torch.zeros_like(c.pages)
    yq = ops.qk_pair_kv4(wide[:, 4:4 + 8 * 128], _dev(c.qn), _dev(c.kn), _dev(c.cos)[None], _dev(c.sin)[None], pages,
                         _dev(c.table), _dev(c.starts), _dev(c.lens))
    assert torch.equal(pages, c.pages) and torch.equal(yq.cpu(), c.yq)


def _attend(rows, ctx, hq, hk, seed, window=0, sinks=0, max_rows=None, lead=0, tail=0, poison=True, scale=128 ** -0.5,
            width=None, table_edit=None):
    table, starts, lens, num = _batch(rows, ctx, hk, seed, width=width, lead=lead)
    if table_edit:
        table_edit(table)
    g = torch.Generator().manual_seed(seed + 7)
    k = torch.randn(num, hk, 64, 128, generator=g, dtype=torch.float64) * 1.3
    v = torch.randn(num, hk, 64, 128, generator=g, dtype=torch.float64) * 0.7
    pages = ref.pack(k, v)
    if poison:  # what no sequence holds is NaN: scales of tokens past the end, whole spare pages
        pages = ref.poison(pages, table, lens)
    total = int(starts[-1]) + tail
    q = (torch.randn(hq, total, 128, generator=g) * 1.5).to(BF16)
    out = torch.full((total, hq, 128), 7.0, dtype=BF16, device=DEV)
    got = ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), scale, window=window,
                            sinks=sinks, max_rows=max_rows, out=out).cpu()
    want, limit = ref.attention(q, pages, table, starts, lens, scale, window, sinks)
    live = slice(int(starts[0]), int(starts[-1]))
    diff, limit = (got.double() - want).abs()[live], limit[live]
    assert torch.isfinite(got.float()[live]).all()
    assert (diff <= limit).all(), f"{(diff / limit).max()} of the bound"
    assert (got[:live.start] == 7).all() and (got[live.stop:] == 7).all()
    return got


@pytest.mark.parametrize("hq,hk", [(4, 1), (8, 8), (16, 8), (5, 1), (16, 2), (12, 1), (40, 2)])
@pytest.mark.parametrize("ctx", [[1], [15, 16, 17, 64], [65, 1, 300], [4097]])
def test_decode(hq, hk, ctx):
    _attend([1] * len(ctx), ctx, hq, hk, seed=hq + len(ctx), max_rows=1, lead=1, tail=2)


@pytest.mark.parametrize("rows,ctx", [([2], [2]), ([5, 1, 0, 3], [70, 1, 40, 64]), ([17], [200]), ([64, 33], [64, 500]),
                                      ([130], [1200]), ([200, 1], [263, 900]), ([8, 6, 1], [300, 77, 1]), ([9, 11], [9, 130])])
@pytest.mark.parametrize("hq,hk", [(4, 1), (4, 4), (16, 2), (3, 1)])
def test_chunks(rows, ctx, hq, hk):
    _attend(rows, ctx, hq, hk, seed=len(rows) + hq, max_rows=max(rows), tail=1)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 0), (64, 3), (100, 64), (128, 130), (5000, 4)])
@pytest.mark.parametrize("rows", [1, 3, 90])
def test_window_and_sinks(rows, window, sinks):
    _attend([rows, rows], [1000, 130], 8, 2, seed=3, window=window, sinks=sinks, max_rows=rows)


@pytest.mark.parametrize("max_rows", [1, 2, 40, None])
def test_max_rows_is_only_a_hint(max_rows):
    _attend([40, 1, 7], [300, 64, 7], 8, 2, seed=9, max_rows=max_rows)


@pytest.mark.parametrize("rows,ctx", [([300, 0, 7, 129], [500, 3, 7, 64]), ([65], [700]), ([64], [64]), ([513, 1], [515, 1300])])
@pytest.mark.parametrize("hint", [5, 8, 9, 64])
def test_long_chunks_with_a_small_hint(rows, ctx, hint):
    """More query tiles than the launch was sized for: a CTA takes several, one or both halves
    of the last, tiles of no key among them."""
    _attend(rows, ctx, 8, 2, seed=31, max_rows=hint, lead=3, tail=2)
    _attend(rows, ctx, 8, 2, seed=32, max_rows=hint, window=70, sinks=5)


def test_more_items_than_processors():
    """Long chunks of many sequences: whole items first, the last wave's cut, some sequences without
    rows or keys."""
    rows, ctx = [64, 70, 0, 64, 1, 130, 64], [640, 70, 40, 300, 0, 1000, 64]
    _attend(rows, ctx, 96, 24, seed=5, max_rows=130, lead=2, tail=3)
    _attend(rows, ctx, 96, 24, seed=6, max_rows=40, window=90, sinks=2)


@pytest.mark.parametrize("seed", range(4))
def test_ragged_batches_share_the_pages(seed):
    """Lengths from nothing to many pages: the runs of pages that the CTAs take cut items anywhere,
    hold many short ones whole, and skip sequences without rows."""
    g = torch.Generator().manual_seed(seed)
    b = [3, 40, 300, 17][seed]
    ctx = [int(x) for x in (torch.rand(b, generator=g) ** 4 * [6000, 1500, 150, 3000][seed]).long()]
    rows = [int(x) for x in torch.randint(0, 3, (b,), generator=g)]
    rows[0] = 1
    _attend(rows, ctx, [8, 8, 2, 24][seed], [2, 1, 1, 2][seed], seed=seed, max_rows=2, lead=1, tail=1)


@pytest.mark.parametrize("b,hk", [(70, 2), (33, 1), (3, 4), (300, 1)])
def test_even_lengths_in_a_wide_table(b, hk):
    """Sequences alike enough that each item is one CTA's, in a table far wider than they need; some
    have no rows, one no keys."""
    g = torch.Generator().manual_seed(b)
    ctx = [int(x) for x in torch.randint(230, 330, (b,), generator=g)]
    rows = [int(x > 0) for x in torch.randint(0, 8, (b,), generator=g)]
    rows[1], ctx[1] = 1, 0
    _attend(rows, ctx, 4 * hk, hk, seed=b, max_rows=1, width=60, lead=1, tail=1)
    _attend(rows, ctx, 12 * hk, hk, seed=b + 1, max_rows=1, width=60, window=100, sinks=3)


@pytest.mark.parametrize("rows,ctx,hq,hk,hint,scale", [
    ([3, 0, 2, 7, 2, 1, 7, 3, 6, 6, 8, 6, 7, 0, 1, 3, 8, 4, 7, 2],
     [278, 28, 93, 12, 387, 27, 7, 21, 6, 81, 48, 22, 123, 6, 28, 15, 19, 326, 31, 108], 8, 8, 2, -0.1),
    ([4, 5, 6, 0, 7, 6, 5, 7, 0, 2, 5, 6, 4, 4, 0, 0, 4, 1, 2, 1],
     [4, 5, 12, 14, 30, 15, 31, 17, 13, 5, 312, 126, 72, 29, 31, 2, 190, 415, 183, 9], 4, 1, 2, 0.3)])
def test_short_ragged_sequences_in_a_wide_table(rows, ctx, hq, hk, hint, scale):
    _attend(rows, ctx, hq, hk, seed=21447, max_rows=hint, width=47, scale=scale, tail=2)


@pytest.mark.parametrize("longest", range(520, 1000, 64))
def test_lengths_at_the_border_of_two_schedules(longest):
    """One sequence longer than the rest by every number of pages around the one where items begin to
    be cut: all CTAs take the same side."""
    rows = [1] * 20
    for other in (64, 130, 200, 260):
        _attend(rows, [longest] + [other] * 19, 8, 8, seed=longest + other, max_rows=1, width=47)
        _attend(rows[:11], [other] * 5 + [longest] + [other + 64] * 5, 4, 1, seed=longest + other, max_rows=1, width=47)


def test_rows_that_see_nothing_are_zero():
    """More rows than the sequence holds: the first of them lie before its start."""
    got = _attend([4, 2], [1, 0], 4, 2, seed=2, max_rows=4)
    assert (got[:3] == 0).all() and (got[3] != 0).any() and (got[4:] == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 30.0])
def test_scales(scale):
    """scale 30 gives scores of thousands: the running maximum has to carry them."""
    _attend([1, 6], [333, 70], 8, 2, seed=4, scale=scale, max_rows=6)
    _attend([1, 20], [333, 70], 8, 2, seed=7, scale=scale, max_rows=20)
    _attend([1, 1, 1], [333, 70, 1], 8, 2, seed=5, scale=scale, max_rows=1)
    _attend([1, 2], [900, 2], 16, 2, seed=6, scale=scale, max_rows=2, window=100, sinks=1)


def test_a_key_that_holds_nearly_all_weight():
    """Large scores: one key's value is most of the result, and where its code is 0 only what the
    offsets' difference leaves of it is."""
    _attend([2, 17, 7, 16, 7, 20], [43, 17, 269, 17, 142, 41], 2, 1, seed=198495, scale=0.3, max_rows=1, width=11)
    _attend([2, 17, 7, 16, 7, 20], [43, 17, 269, 17, 142, 41], 8, 1, seed=198496, scale=0.3, max_rows=20)


def test_queries_of_any_size():
    """Columns from tiny to huge next to each other, with elements far below their column's largest:
    queries are scaled per column for the tensor core."""
    hk, hq = 1, 8
    g = torch.Generator().manual_seed(0)
    pages = ref.pack(*(torch.randn(5, hk, 64, 128, generator=g, dtype=torch.float64) for _ in range(2)))
    q = torch.randn(hq, 1, 128, generator=g) * torch.logspace(-30, 6, hq)[:, None, None]
    q[:, :, ::3] *= 2.0 ** -20
    q[3] = 0
    q = q.to(BF16)
    table = torch.arange(5, dtype=torch.int32)[None]
    starts, lens = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([300], dtype=torch.int32)
    got = ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), 0.05).cpu()
    want, limit = ref.attention(q, pages, table, starts, lens, 0.05, 0, 0)
    assert ((got.double() - want).abs() <= limit).all()


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_nan_reaches_only_the_rows_that_see_it(rows):
    """A key or value that reads as NaN: rows that see it are NaN (the whole row, or the value's
    scale group), rows before it or past the window are exact."""
    hk, hq, n = 1, 4, 200
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(4, hk, 64, 128, generator=g, dtype=torch.float64) for _ in range(2))
    clean = ref.pack(k, v)
    table = torch.arange(4, dtype=torch.int32)[None]
    q = torch.randn(hq, rows, 128, generator=g).to(BF16)
    starts, lens = torch.tensor([0, rows], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    at = n - 1 - rows // 2  # seen by the last rows only
    for base in (8192, 8704):
        pages = clean.clone()
        sc = pages[at // 64, 0, base + 8 * (at % 64):base + 8 * (at % 64) + 2]
        sc.copy_(torch.tensor([0xC0, 0x7F], dtype=torch.uint8))
        got = ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), 0.1, max_rows=rows).cpu()
        want, limit = ref.attention(q, clean, table, starts, lens, 0.1, 0, 0)
        before = rows - 1 - rows // 2  # rows whose position lies before `at`
        assert ((got.double() - want).abs() <= limit)[:before].all()
        assert got[before:, :, :32].isnan().all()
        got = ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), 0.1, max_rows=rows,
                                window=max(1, rows // 2)).cpu()
        want, limit = ref.attention(q, clean, table, starts, lens, 0.1, max(1, rows // 2), 0)
        far = torch.arange(n - rows, n) - at  # distance of each row's position from the poisoned key
        free = (far < 0) | (far >= max(1, rows // 2))
        assert ((got.double() - want).abs() <= limit)[free].all() and got[~free][:, :, :32].isnan().all()


def test_growing_scores_move_the_maximum():
    """Keys whose scores climb over the context make every tile rescale."""
    hk, n = 1, 8
    table = torch.arange(n, dtype=torch.int32)[None]
    ramp = torch.linspace(0, 4, n * 64, dtype=torch.float64).reshape(n, 1, 64, 1)
    g = torch.Generator().manual_seed(0)
    k = ramp * torch.ones(128, dtype=torch.float64)
    v = torch.randn(n, hk, 64, 128, generator=g, dtype=torch.float64)
    pages = ref.pack(k, v)
    q = torch.ones(4, 1, 128).to(BF16)
    starts, lens = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([n * 64], dtype=torch.int32)
    got = ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), 1.0).cpu()
    want, limit = ref.attention(q, pages, table, starts, lens, 1.0, 0, 0)
    assert ((got.double() - want).abs() <= limit).all()


def test_shared_prefix_pages_and_wide_table():
    def share(table):
        table[1, :2] = table[0, :2]
        table[2, :1] = table[0, :1]

    _attend([1, 2, 1], [200, 140, 70], 8, 2, seed=6, max_rows=2, width=40, table_edit=share)


def test_bad_pages_are_left_out():
    """Ids outside the cache are not dereferenced: their keys are left out, reads give zeros, and
    the device error word says so."""
    hk, hq = 2, 4
    table = torch.tensor([[0, -1, 2, 99]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    pages = ref.pack(*(torch.randn(3, hk, 64, 128, generator=g, dtype=torch.float64) for _ in range(2)))
    q = torch.randn(hq, 1, 128, generator=g).to(BF16)
    starts, lens = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([250], dtype=torch.int32)
    got = ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), 0.1).cpu()
    assert L.device_error(clear=True) == 1 << 5
    whole = torch.tensor([[0, 2]], dtype=torch.int32)
    want, limit = ref.attention(q, pages, whole, starts, torch.tensor([128], dtype=torch.int32), 0.1, 0, 0)
    assert ((got.double() - want).abs() <= limit).all()
    before = _dev(pages)
    after = before.clone()
    qkv = torch.randn(4, (hq + 2 * hk) * 128, generator=g).to(BF16)
    table = torch.tensor([[0, -1]], dtype=torch.int32)
    starts, lens = torch.tensor([0, 4], dtype=torch.int32), torch.tensor([130], dtype=torch.int32)
    cos = torch.ones(4, 128, dtype=BF16)
    ops.qk_pair_kv4(_dev(qkv), _dev(_norm(1)), _dev(_norm(2)), _dev(cos), _dev(cos), after, _dev(table), _dev(starts), _dev(lens))
    assert torch.equal(before, after) and L.device_error(clear=True) == 1 << 5
    k, v = ops.kv4_read(before, _dev(table), _dev(starts), _dev(lens), 4)
    assert not k.any() and not v.any() and L.device_error(clear=True) == 1 << 5


def test_context_longer_than_the_table():
    table = torch.tensor([[1]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    pages = ref.pack(*(torch.randn(2, 1, 64, 128, generator=g, dtype=torch.float64) for _ in range(2)))
    q = torch.randn(4, 1, 128, generator=g).to(BF16)
    starts, lens = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([100], dtype=torch.int32)
    got = ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), 0.1).cpu()
    assert L.device_error(clear=True) == 1 << 5
    want, limit = ref.attention(q, pages, table, starts, torch.tensor([64], dtype=torch.int32), 0.1, 0, 0)
    assert ((got.double() - want).abs() <= limit).all()


def test_decoding_steps_in_a_captured_graph():
    """Steps as they are used: write, then attend, captured once and replayed while the lengths
    grow on the device; every step equals the plain formula over what the cache holds."""
    hq, hk, b = 8, 2, 3
    ctx = torch.tensor([62, 1, 130], dtype=torch.int32)
    table = torch.arange(b * 4, dtype=torch.int32).reshape(b, 4).flip(1).contiguous()
    pages = ops.kv4_pages(b * 4, hk)
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(b * 4, hk, 64, 128, generator=g, dtype=torch.float64) for _ in range(2))
    pages.copy_(ref.pack(k, v))
    qkv = torch.zeros(b, (hq + 2 * hk) * 128, dtype=BF16, device=DEV)
    cos, sin = torch.zeros(b, 128, dtype=BF16, device=DEV), torch.zeros(b, 128, dtype=BF16, device=DEV)
    qn, kn = _norm(1), _norm(2)
    starts, lens, tab = torch.arange(b + 1, dtype=torch.int32, device=DEV), ctx.to(DEV), table.to(DEV)
    dq, dk = _dev(qn), _dev(kn)

    def step():
        yq = ops.qk_pair_kv4(qkv, dq, dk, cos, sin, pages, tab, starts, lens)
        return yq, ops.attention_kv4(yq, pages, tab, starts, lens, 128 ** -0.5, max_rows=1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, out = step()
    for i in range(4):
        lens.add_(1)
        qkv.copy_(torch.randn(b, (hq + 2 * hk) * 128, generator=g).to(BF16))
        angle = torch.rand(b, 128, generator=g)
        cos.copy_(angle.cos().to(BF16))
        sin.copy_(angle.sin().to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        want, limit = ref.attention(yq.cpu(), pages.cpu(), table, starts.cpu(), lens.cpu(), 128 ** -0.5, 0, 0)
        q, kk, vv = ref.norm_rotate_quantize(qkv.cpu(), qn, kn, cos.cpu(), sin.cpu(), hq, hk)
        gk, gv = ops.kv4_read(pages, tab, starts, lens, b)
        assert torch.equal(gk.cpu().double(), kk) and torch.equal(gv.cpu().double(), vv)
        assert ((out.cpu().double() - want).abs() <= limit).all()


def _long_cache(rows, hq, hk, seed):
    table, starts, lens, num = _batch([rows, rows], [3000, 700], hk, seed)
    g = torch.Generator().manual_seed(seed)
    pages = _dev(ref.pack(*(torch.randn(num, hk, 64, 128, generator=g, dtype=torch.float64) for _ in range(2))))
    q = torch.randn(hq, 2 * rows, 128, generator=g).to(BF16).to(DEV)
    return q, (pages, _dev(table), _dev(starts), _dev(lens))


@pytest.mark.parametrize("rows", [1, 40])
def test_another_stream_and_two_calls_at_once(rows):
    q, place = _long_cache(rows, 8, 2, 13)
    first = ops.attention_kv4(q, *place, 0.1, max_rows=rows)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(5):
                outs.append(ops.attention_kv4(q, *place, 0.1, max_rows=rows))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("rows", [1, 40])
def test_captured_calls_with_workspaces(rows):
    """Shares of long sequences joined in a replayed graph, the lengths changed between replays, two
    graphs at once on two streams."""
    q, place = _long_cache(rows, 8, 2, 14)
    lens = place[3]
    ops.attention_kv4(q, *place, 0.1, max_rows=rows)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.attention_kv4(q, *place, 0.1, max_rows=rows))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for grow in (0, -37, 20, -400):
        lens.add_(grow)
        want = ops.attention_kv4(q, *place, 0.1, max_rows=rows)
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("rows", [1, 100])
def test_first_call_of_a_process_is_captured(rows):
    """Nothing that a call sets up once (attributes, symbols, modules) disturbs a capture."""
    code = f"""
import torch
from fastforward_b200 import ops
pages = ops.kv4_pages(8, 2)
table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
starts = torch.tensor([0, {rows}], dtype=torch.int32, device="cuda")
lens = torch.tensor([300], dtype=torch.int32, device="cuda")
q = torch.randn(8, {rows}, 128, device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.attention_kv4(q, pages, table, starts, lens, 0.1)
    k, v = ops.kv4_read(pages, table, starts, lens, {rows})
graph.replay()
torch.cuda.synchronize()
assert (y == 0).all() and (k == 0).all() and (v == 0).all()
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=Path(__file__).resolve().parents[1])


def test_pages_past_32_bits():
    """A cache of more than 2^32 bytes: pages at its far end."""
    hk, hq, num = 8, 8, 60000
    pages = torch.empty(num, hk, L.KV4_RECORD, dtype=torch.uint8, device=DEV)
    g = torch.Generator().manual_seed(3)
    few = ref.pack(*(torch.randn(3, hk, 64, 128, generator=g, dtype=torch.float64) for _ in range(2)))
    far = [num - 1, num - 2, num - 7]
    for i, p in enumerate(far):
        pages[p] = few[i].to(DEV)
    q = torch.randn(hq, 1, 128, generator=g).to(BF16)
    starts, lens = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([150], dtype=torch.int32)
    got = ops.attention_kv4(_dev(q), pages, torch.tensor([far], dtype=torch.int32, device=DEV), _dev(starts), _dev(lens), 0.1).cpu()
    want, limit = ref.attention(q, few, torch.tensor([[0, 1, 2]], dtype=torch.int32), starts, lens, 0.1, 0, 0)
    assert ((got.double() - want).abs() <= limit).all()


def test_empty_call():
    pages = ops.kv4_pages(1, 2)
    z = torch.zeros(2, dtype=torch.int32, device=DEV)
    q = torch.zeros(4, 0, 128, dtype=BF16, device=DEV)
    out = ops.attention_kv4(q, pages, z[:1, None], z, z[:1], 0.1)
    assert out.shape == (0, 4, 128)
