"""Edges of the 4-bit K/V cache on the GPU: values at both ends of what is held, NaN, absent
pages in every schedule, and each kernel within a bound of its own arithmetic."""
import types

import pytest
import torch

from fastforward_b200 import _lib as L
from fastforward_b200 import ops
from tests import _kv4 as ref
from tests import _kv4_bounds as bounds

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(clear=True)
    yield
    assert L.device_error(clear=True) == 0


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def _norm(seed, eps=1e-6):
    g = torch.Generator().manual_seed(seed)
    return types.SimpleNamespace(weight=(1 + 0.2 * torch.randn(128, generator=g)).to(BF16), variance_epsilon=eps)


def _dev(x):
    if isinstance(x, types.SimpleNamespace):
        return types.SimpleNamespace(weight=x.weight.to(DEV), variance_epsilon=x.variance_epsilon)
    return x.to(DEV)


def _run(q, pages, table, starts, lens, scale, **kw):
    return ops.attention_kv4(_dev(q), _dev(pages), _dev(table), _dev(starts), _dev(lens), scale, **kw).cpu()


def _kv(num, hk, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(num, hk, 64, 128, generator=g, dtype=torch.float64) for _ in range(2))


@pytest.mark.parametrize("rows", [40, 640])
@pytest.mark.parametrize("eps", [1e-6, 0.0, 1e-30, 3.0])
def test_written_queries_of_any_size(rows, eps):
    """Rows from tiny to huge, past where fp32 holds their squares' sum: the queries are the formula's."""
    hq, hk = 4, 1
    g = torch.Generator().manual_seed(rows)
    qkv = (torch.randn(rows, (hq + 2 * hk) * 128, generator=g) * torch.logspace(-37, 37, rows)[:, None]).to(BF16)
    qkv[7, :128:3] = (qkv[7, :128:3].double() * 2.0 ** -40).to(BF16)
    angle = torch.rand(rows, 128, generator=g) * 6.3
    cos, sin = angle.cos().to(BF16), angle.sin().to(BF16)
    qn, kn = _norm(1, eps), _norm(2, eps)
    pages = ops.kv4_pages(rows // 64 + 1, hk)
    table = torch.arange(pages.shape[0], dtype=torch.int32)[None]
    got = ops.qk_pair_kv4(_dev(qkv), _dev(qn), _dev(kn), _dev(cos), _dev(sin), pages, _dev(table), _dev(_ints(0, rows)),
                          _dev(_ints(rows))).cpu().double()
    # eps is a float in the call.  Sixteen roundings of fp32 at most (sum of squares, half of each; root,
    # products) on each of two terms and one to bf16, of
    # which the smallest number is 2^-133
    exact = types.SimpleNamespace(weight=qn.weight, variance_epsilon=float(torch.tensor(eps, dtype=torch.float32)))
    want = ref.norm_rotate(qkv.double().reshape(rows, -1, 128).transpose(0, 1)[:hq], exact, cos, sin)
    terms = ref.query_terms(qkv, exact, cos, sin, hq)
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + terms * 2.0 ** -20 + 2.0 ** -134).all()


def _group_nan(pages, page, token, value):
    """The first scale group of a token of head 0 reads as NaN: its key (value 0) or its value (1)."""
    at = 8192 + 512 * value + 8 * token
    pages[page, 0, at:at + 2] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8)


@pytest.mark.parametrize("value", [0, 1])
@pytest.mark.parametrize("rows,n,at,low", [(1, 70, 66, (66, 67)), (1, 70, 3, (3, 4)), (3, 70, 64, (60, 67)),
                                           (40, 90, 66, (66, 67)), (1, 6000, 100, (0, 1500)), (1, 6000, 4000, (3000, 4500)),
                                           (40, 6000, 100, (0, 1500))])
def test_nan_of_no_weight_is_seen(value, rows, n, at, low):
    """A key or value that reads as NaN, beside keys `low` whose probability is 0 in fp32, its own
    among them: 0 x NaN is NaN in the rows that see it, whatever page, CTA or kernel it falls to."""
    num = -(-n // 64)
    k, v = _kv(num, 1, 3)
    for j in range(*low):
        k[j // 64, :, j % 64] = -8.0
    pages = ref.pack(k, v)
    _group_nan(pages, at // 64, at % 64, value)
    q = torch.ones(4, rows, 128).to(BF16)  # scores of the low keys: -1024
    table = torch.arange(num, dtype=torch.int32)[None]
    for width in (num, 200):  # narrow: an item a CTA; wide: shared out
        wide = torch.full((1, max(width, num)), -1, dtype=torch.int32)
        wide[:, :num] = table
        got = _run(q, pages, wide, _ints(0, rows), _ints(n), 1.0, max_rows=rows)
        sees = torch.arange(n - rows, n) >= at
        assert got[sees][..., :32].isnan().all()
        assert not got[~sees].isnan().any()


@pytest.mark.parametrize("rows", [1, 4, 40])
@pytest.mark.parametrize("scale,size", [(2.0 ** 100, 2.0 ** 20), (2.0 ** 60, 2.0 ** 60), (1.0, 2.0 ** 115), (2.0 ** 120, 1.0),
                                        (0.7, 2.0 ** 80), (0.09, 2.0 ** 40), (-0.3, 2.0 ** 30), (2.0 ** 25, 1.0)])
@pytest.mark.parametrize("ctx", [250, 5000])
@pytest.mark.parametrize("below", [False, True])
def test_scores_past_what_exp2_can_tell(rows, scale, size, ctx, below):
    """Scores of 2^25 to 2^123, of both signs or all below 0: next to the best key the others have no
    weight, so each row is that key's value, whatever queries and scale the size comes from."""
    num = -(-ctx // 64)
    k, v = _kv(num, 1, 8)
    q = torch.randn(4, rows, 128, generator=torch.Generator().manual_seed(5)) * size
    if below:
        k, q = k.abs(), -q.abs() if scale > 0 else q.abs()
    pages, q = ref.pack(k, v), q.to(BF16)
    got = _run(q, pages, torch.arange(num, dtype=torch.int32)[None], _ints(0, rows), _ints(ctx), scale, max_rows=rows).double()
    held_k, held_v = (x.reshape(num * 64, 128) for x in ref.unpack(pages))
    s = q.double() @ held_k.T * scale
    s.masked_fill_(torch.arange(num * 64) > torch.arange(ctx - rows, ctx)[:, None], -torch.inf)
    best = s.topk(2, -1)
    clear = best.values[..., 0] - best.values[..., 1] > 100 + 2.0 ** -15 * best.values[..., 0].abs()  # fp32 products tell them apart
    assert clear.double().mean() > 0.9
    want = held_v[best.indices[..., 0]]
    # the offsets leave 2^-22 255 of the scale of the value's group, below 2^-14 of the row's largest
    off = (got.transpose(0, 1) - want).abs() <= want.abs() * 2.0 ** -8 * 2.02 + 2.0 ** -14 * want.abs().amax(-1, keepdim=True)
    assert off[clear].all()


def test_outputs_in_place_of_their_inputs():
    """One row, or one head: the layouts of queries and result agree and the result may replace them."""
    k, v = _kv(60, 2, 5)
    pages, table = ref.pack(k, v), torch.arange(60, dtype=torch.int32)[None]
    g = torch.Generator().manual_seed(1)
    for hq, rows, hk in ((8, 1, 2), (96, 1, 2), (1, 20, 1), (1, 300, 1)):
        q = _dev(torch.randn(hq, rows, 128, generator=g).to(BF16))
        place = (_dev(pages[:, :hk].contiguous()), _dev(table), _dev(_ints(0, rows)), _dev(_ints(3800)))
        want = ops.attention_kv4(q, *place, 0.1)
        got = ops.attention_kv4(q, *place, 0.1, out=q.view(rows, hq, 128))
        assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    q = _dev(torch.randn(4, 6, 128, generator=g).to(BF16))
    with pytest.raises(ValueError, match="overlap"):
        ops.attention_kv4(q, *place[:2], _dev(_ints(0, 6)), place[3], 0.1, out=q.view(6, 4, 128))
    both = torch.zeros(4 * 6 * 128 + 64, dtype=BF16, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ops.attention_kv4(both[:-64].view(4, 6, 128), *place[:2], _dev(_ints(0, 6)), place[3], 0.1, out=both[64:].view(6, 4, 128))


def test_written_queries_in_place_of_one_row():
    g = torch.Generator().manual_seed(2)
    cos, sin = (_dev(torch.rand(3, 128, generator=g).to(BF16)) for _ in range(2))
    qn, kn = _dev(_norm(1)), _dev(_norm(2))
    for rows in (1, 3):
        qkv = _dev(torch.randn(rows, 8 * 128, generator=g).to(BF16))
        pages = [ops.kv4_pages(1, 2) for _ in range(2)]
        place = (_dev(_ints(0))[None], _dev(_ints(0, rows)), _dev(_ints(rows)))
        want = ops.qk_pair_kv4(qkv, qn, kn, cos[:rows], sin[:rows], pages[0], *place)
        into = qkv.view(-1)[:4 * rows * 128].view(4, rows, 128)
        if rows == 1:
            got = ops.qk_pair_kv4(qkv, qn, kn, cos[:rows], sin[:rows], pages[1], *place, out=into)
            assert torch.equal(got, want) and torch.equal(*pages)
        else:
            with pytest.raises(ValueError, match="overlap"):
                ops.qk_pair_kv4(qkv, qn, kn, cos[:rows], sin[:rows], pages[1], *place, out=into)


@pytest.mark.parametrize("rows", [1, 4, 40])
@pytest.mark.parametrize("power", [-90, -62, -40, 40, 54])
@pytest.mark.parametrize("ctx", [70, 5000])
def test_values_at_both_ends_of_the_range(rows, power, ctx):
    """Values from the largest that attention takes to the smallest that the cache holds, through both kernels:
    the one for few columns holds its sums to 2^-80 only."""
    num = -(-ctx // 64)
    k, v = _kv(num, 2, power + 100)
    v = v.clamp(-3.5, 3.5) * 2.0 ** power  # below 2^57, above 2^-100 for the most part
    pages, table = ref.pack(k, v), torch.arange(num, dtype=torch.int32)[None]
    q = torch.randn(8, rows, 128, generator=torch.Generator().manual_seed(2)).to(BF16)
    got = _run(q, pages, table, _ints(0, rows), _ints(ctx), 0.1, max_rows=rows).double()
    want, limit = bounds.attention(q, pages, table, _ints(0, rows), _ints(ctx), 0.1, registers=rows * 4 <= 32)
    assert ((got - want).abs() <= limit).all()


@pytest.mark.parametrize("rows,hq,hk,ctx,width,hint", [
    (1, 8, 2, [250], 4, 1),                        # an item a CTA
    (1, 8, 2, [3000, 2000, 1500], 60, 1),          # equal runs that cut the items
    (3, 8, 2, [4000, 64, 900], 70, 3),
    (1, 8, 2, [250, 300, 260, 200], 60, 1),        # items apart in a wide table
    (40, 8, 2, [2500], 40, 40),                    # tcgen05, in shares
    (20, 16, 2, [700, 130, 64, 900], 16, 20),
    (80, 96, 24, [400, 300, 500, 200], 9, 80),     # tcgen05, whole items and shares
    (70, 8, 2, [600, 200], 12, 9),                 # more items than the launch was sized for
])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 70)])
def test_absent_pages_in_every_schedule(rows, hq, hk, ctx, width, hint, window, sinks):
    """Ids outside the cache, in both halves of a block of two pages and in first and last pages of items:
    their keys are left out.  The ids point just past the slice that the call is given, where
    pages of NaN lie."""
    b = len(ctx)
    need = [-(-c // 64) for c in ctx]
    num = sum(need)
    k, v = _kv(num, hk, rows + b)
    pages = ref.pack(k, v)
    table = torch.full((b, width), num + 1, dtype=torch.int32)
    order = torch.randperm(num, generator=torch.Generator().manual_seed(rows)).to(torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
        absent = {2: [0], 1: []}.get(n, [2, 3] if n < 6 else [0, 3, 6, 7, n - 2] + list(range(9, n - 3, 5)))
        for j in absent:
            if j < n - 1:
                table[i, j] = [num, -1, num + 2, -2 ** 31, 2 ** 31 - 1][j % 5]
    if b > 1:
        table[1, need[1] - 1] = num  # the newest keys
    starts, lens = torch.arange(b + 1, dtype=torch.int32) * rows, _ints(*ctx)
    q = torch.randn(hq, b * rows, 128, generator=torch.Generator().manual_seed(7)).to(BF16)
    more = torch.cat([pages, torch.full((4, hk, L.KV4_RECORD), 0xFF, dtype=torch.uint8)])
    got = ops.attention_kv4(_dev(q), _dev(more)[:num], _dev(table), _dev(starts), _dev(lens), 0.1, window=window, sinks=sinks,
                            max_rows=hint).cpu().double()
    assert L.device_error(clear=True) == 1 << 5
    want, limit = bounds.attention(q, pages, table, starts, lens, 0.1, window, sinks, registers=hint * hq // hk <= 32)
    assert ((got - want).abs() <= limit).all()


@pytest.mark.parametrize("rows,ctx,hint", [(1, 200, 1), (1, 5000, 1), (40, 200, 40), (40, 5000, 40), (150, 2600, 9)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 3)])
def test_contexts_past_the_table(rows, ctx, hint, window, sinks):
    """Positions from the table's width on are left out, whole rows among them."""
    for held in (ctx // 2, ctx - 65):
        if held < 64:
            continue
        num = held // 64
        k, v = _kv(num, 2, rows)
        pages, table = ref.pack(k, v), torch.arange(num, dtype=torch.int32)[None]
        q = torch.randn(8, rows, 128, generator=torch.Generator().manual_seed(3)).to(BF16)
        more = torch.cat([_dev(table), torch.zeros(1, 400, dtype=torch.int32, device=DEV)], 1)[:, :num]
        got = ops.attention_kv4(_dev(q), _dev(pages), more, _dev(_ints(0, rows)), _dev(_ints(ctx)), 0.1, window=window,
                                sinks=sinks, max_rows=hint).cpu().double()
        assert L.device_error(clear=True) == 1 << 5
        want, limit = bounds.attention(q, pages, table, _ints(0, rows), _ints(ctx), 0.1, window, sinks, registers=hint * 4 <= 32)
        assert ((got - want).abs() <= limit).all()


@pytest.mark.parametrize("rows,hq,hk,ctx,hint", [
    (1, 4, 2, [40000], 1), (4, 16, 2, [9000, 30], 4), (1, 300, 1, [500, 70], 1), (1, 1, 1, [20000] * 3, 1),
    (40, 8, 2, [9000], 40), (300, 4, 4, [700, 3000], 300), (33, 1, 1, [33, 6000], 33)])
def test_each_kernel_within_its_own_bound(rows, hq, hk, ctx, hint):
    """Long contexts, where the sums' own rounding counts, and wide groups; the kernel of more than 32
    columns multiplies values without an offset and is held to that."""
    need = [-(-c // 64) for c in ctx]
    k, v = _kv(sum(need), hk, 17)
    pages = ref.pack(k, v + 0.5)  # sums that grow
    table = torch.zeros(len(ctx), max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.arange(at, at + n)
        at += n
    starts, lens = torch.arange(len(ctx) + 1, dtype=torch.int32) * rows, _ints(*ctx)
    q = torch.randn(hq, len(ctx) * rows, 128, generator=torch.Generator().manual_seed(4)).to(BF16)
    got = _run(q, pages, table, starts, lens, 0.088, max_rows=hint).double()
    want, limit = bounds.attention(q, pages, table, starts, lens, 0.088, registers=hint * hq // hk <= 32)
    assert ((got - want).abs() <= limit).all()


def test_a_write_of_more_rows_than_a_grid_is_high():
    """70000 rows: the launch's rows need its third dimension."""
    rows = 70000
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(rows, 3 * 128, generator=g).to(BF16)
    angle = torch.rand(rows, 128, generator=g) * 6.3
    cos, sin = angle.cos().to(BF16), angle.sin().to(BF16)
    qn, kn = _norm(1), _norm(2)
    pages = ops.kv4_pages(-(-rows // 64), 1)
    place = (torch.arange(pages.shape[0], dtype=torch.int32, device=DEV).flip(0)[None].contiguous(), _dev(_ints(0, rows)), _dev(_ints(rows)))
    yq = ops.qk_pair_kv4(_dev(qkv), _dev(qn), _dev(kn), _dev(cos), _dev(sin), pages, *place).cpu().double()
    gk, gv = (x.cpu().double() for x in ops.kv4_read(pages, *place, rows))
    q, k, v = ref.norm_rotate_quantize(qkv, qn, kn, cos, sin, 1, 1)
    assert torch.equal(gk, k) and torch.equal(gv, v)
    assert ((yq - q).abs() <= q.abs() * 2.0 ** -8 * 1.01 + ref.query_terms(qkv, qn, cos, sin, 1) * 2.0 ** -20).all()


@pytest.mark.parametrize("active", [(0, 999), (3, 4, 500, 998), (999,), (0, 1, 2, 700, 701, 997), tuple(range(0, 1000, 37))])
@pytest.mark.parametrize("hq,hk,hint", [(8, 2, 1), (12, 1, 3), (80, 2, 1)])
def test_few_active_sequences_among_a_thousand(active, hq, hk, hint):
    """Slots without rows between those with some, at a run's borders too; their contexts do not matter."""
    b, rows, ctx = 1000, [0] * 1000, [77] * 1000
    for j, i in enumerate(active):
        rows[i], ctx[i] = 1 + j % 3, 5 + 611 * (j % 5) + j
    num = sum(-(-ctx[i] // 64) for i in active)
    table = torch.full((b, 41), -1, dtype=torch.int32)
    at = 0
    for i in active:
        n = -(-ctx[i] // 64)
        table[i, :n] = torch.arange(at, at + n)
        at += n
    k, v = _kv(num, hk, 12)
    pages = ref.pack(k, v)
    starts, lens = _ints(0, *torch.tensor(rows).cumsum(0).tolist()), _ints(*ctx)
    q = torch.randn(hq, sum(rows), 128, generator=torch.Generator().manual_seed(6)).to(BF16)
    got = _run(q, pages, table, starts, lens, 0.1, max_rows=min(hint, sum(rows))).double()
    want, limit = bounds.attention(q, pages, table, starts, lens, 0.1, registers=min(hint, sum(rows)) * hq // hk <= 32)
    assert ((got - want).abs() <= limit).all()


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_equal_scores_where_they_become_vast(rows):
    """Two keys of the same score, 2^30 + 48 in base 2, next to which nothing else counts: one is the first that
    its warps see, one comes after scores of -2^32.  Each has half the weight."""
    k = torch.full((8, 1, 64, 128), -28.0, dtype=torch.float64)
    k[1, 0, 3] = k[4, 0, 5] = 7.0
    _, v = _kv(8, 1, 9)
    pages = ref.pack(k, v)
    q = torch.ones(4, rows, 128).to(BF16)
    near = torch.arange(-64, 64).to(torch.float32) / 16 + 830648.625
    scale = float(near[(near * torch.tensor(1.4426950408889634)).double() == 1198372.625][0])  # 896 times that: the score
    table = torch.arange(8, dtype=torch.int32)[None]
    for width in (8, 100):
        wide = torch.nn.functional.pad(table, (0, width - 8), value=-1)
        got = _run(q, pages, wide, _ints(0, rows), _ints(500), scale, max_rows=rows).double()
        held = ref.unpack(pages)[1][:, 0]
        want, most = (held[1, 3] + held[4, 5]) / 2, torch.maximum(held[1, 3].abs(), held[4, 5].abs())
        # a probability's and the result's rounding, and the offsets' 2^-22 255 of a scale
        assert ((got - want).abs() <= (2 * most + want.abs()) * 2.0 ** -8 * 1.01 + 2.0 ** -14 * most.amax()).all()
