"""The paged cache's attention: limits of its number formats, and every form of its kernels on purpose.

A form is told from outside by the workspace that a call asks for: 520 bytes a row of a partial result, in 16- or 32-row
columns for the streaming form, 256 rows for the tile form, two for every compute unit where all tiles are shared evenly."""
import ctypes
import math

import pytest
import torch

from oracle import kv_cache as okv
from test_gpu_kv_cache import PAGES, Case, ManyRows, Pool

pytestmark = pytest.mark.gpu

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _weights(case, h, row):
    """(p_j 2^e_j at its largest, sum_j |code_j| of every element) of packed row `row`, query head h, one sequence, group 1,
    no mask."""
    n, page = case.lens[0], case.page
    at = torch.tensor(case.table[0])[torch.arange(n) // page]
    k = okv.values(case.host["k"], case.host["k_scale"])[at, h, torch.arange(n) % page]
    codes = okv.values(case.host["v"], torch.zeros_like(case.host["v_scale"]))[at, h, torch.arange(n) % page]
    p = torch.softmax(case.q[row, h].double() @ k.T / math.sqrt(128), -1)
    e = case.host["v_scale"][at, h].double()
    return (p * torch.exp2(e)).max(), codes.abs().sum(0)


@pytest.mark.parametrize("kind,half", [(Case, 2.0 ** -39), (ManyRows, None)])
@pytest.mark.parametrize("page", (16, 32, 64, 128))
@pytest.mark.parametrize("apart", [0, 12, 24, 34, 40, 96])
def test_weights_far_below_the_largest(dev, kind, half, page, apart):
    """Every other page has zero codes and a scale 2^apart as large.  The weights of the others' tokens are that much smaller
    than the largest, and fp16 keeps 2^-25 of its unit: 2^-39 of the largest weight in the streaming form (unit 2^14), 2^-33
    in the tile form (2^8), twice that where weights are rounded again.  That, times the codes, comes on top of the bound
    of the other tests, and is nothing while scales are 2^12 apart."""
    half = half or (2.0 ** -33 if page >= 64 else 2.0 ** -32)
    c = kind(dev, [4], [8 * page], heads=2, page=page, seed=apart + page)
    for i, at in enumerate(c.table[0]):
        c.host["v_scale"][at] = 48 - apart if i % 2 == 0 else 48
        if i % 2:
            c.host["v"].view(torch.uint8)[at] = 0
    c.cache.v.view(torch.uint8).copy_(c.host["v"].view(torch.uint8))
    c.cache.v_scale.view(torch.uint8).copy_((c.host["v_scale"] + 127).to(torch.uint8))
    got = c.attend(causal=False).double().cpu()
    want, size = c.want(causal=False)
    for row in range(4):
        for h in range(2):
            top, codes = _weights(c, h, row)
            most = 2.0 ** -8 * want[row, h].abs() + 2.0 ** -9 * size[row, h]
            if apart > 12:
                most += half * top * codes
            assert ((got[row, h] - want[row, h]).abs() <= most).all(), (row, h)


# ------------------------------------------------------------------------------------------------ forms

def workspace(cache, plan, q, window=0):
    from diffsynth_engine_amd import _lib

    P = _lib.KVAttnParams(total_rows=q.shape[0], softmax_scale=0.1, heads_q=q.shape[1], window=window)
    return _lib.load().dsx_kv_attn_workspace_bytes(cache._ref, plan._ref, ctypes.byref(P))


def agree(a, b, pool, plan, q, **kw):
    """Two results of the same call, each within 2^-8 |o| + 2^-9 A of the exact one (the bound of the other tests), where
    A = sum_j p_j |v_j| is the same attention over the codes' magnitudes."""
    from diffsynth_engine_amd import kv_cache, ops

    sizes = pool.codes[1].view(torch.uint8).bitwise_and(0x7f).view(F8)
    cache = kv_cache.KVCache(pool.cache.k, sizes, pool.cache.k_scale, pool.cache.v_scale)
    size = ops.kv_attention(q, cache, plan, split_keys=False, **kw).double()
    off = (a.double() - b.double()).abs() - 2.0 ** -7 * (1 + 2.0 ** -6) * b.double().abs() - 2.0 ** -8 * (1 + 2.0 ** -6) * size
    assert off.max().item() <= 0, off.max().item()


def compute_units(dev):
    return torch.cuda.get_device_properties(dev).multi_processor_count


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("batch,heads,group,rows", [
    (66, 8, 4, 1),     # one column of 16 rows
    (66, 8, 4, 5),     # two: 20 of 32
    (50, 8, 1, 32),    # all 32, and sequences of 16 and fewer among them
    (700, 8, 17, 1),   # one row in the second column; more sequences than lanes; several units a share
    (1, 40, 7, 4),     # a share is a piece of one unit
])
def test_even_shares(dev, page, batch, heads, group, rows):
    from diffsynth_engine_amd import ops

    g = torch.Generator().manual_seed(batch + rows)
    top = {1: 150000, 700: 1024}.get(batch, 16384)
    pool = Pool(dev, heads, 64, page, seed=batch + page)
    lens = torch.randint(0, top + 1, (batch,), generator=g).tolist()
    lens[-1], lens[batch // 2] = top, top - 17
    count = [min(int(r), n) for r, n in zip(torch.randint(0, rows + 1, (batch,), generator=g), lens)]
    count[-1] = count[batch // 2] = rows
    plan, starts, table, q = pool.batch(count, lens, group)
    cus = compute_units(dev)
    columns = 1 if rows * group <= 16 else 2
    some = sorted({0, batch // 2, batch - 1} | set(range(3, batch, max(batch // 5, 1))))
    for kw in (dict(), dict(window=top - top // 5), dict(causal=False)):
        assert batch * heads * ((top - top // 5 if "window" in kw else top) // 32) >= 512 * cus
        assert workspace(pool.cache, plan, q, kw.get("window", 0)) == 2 * cus * 16 * columns * 520
        out = torch.full_like(q, 7.0)
        ops.kv_attention(q, pool.cache, plan, out=out, **kw)
        pool.check(out, q, starts, table, lens, only=some, **kw)
        assert not out.isnan().any() and torch.equal(out, ops.kv_attention(q, pool.cache, plan, **kw))
        whole = ops.kv_attention(q, pool.cache, plan, split_keys=False, **kw)  # every sequence, against the other form
        agree(out, whole, pool, plan, q, **kw)


@pytest.mark.parametrize("page", (16, 64))
def test_even_shares_of_what_breaks_a_bound(dev, page):
    from diffsynth_engine_amd import ops

    pool = Pool(dev, 8, 64, page, seed=3)
    lens = [16384, 9000, 0, 16000] * 17
    plan, starts, table, q = pool.batch([5, 3, 2, 4] * 17, lens, 4)
    assert workspace(pool.cache, plan, q) == 2 * compute_units(dev) * 32 * 520
    clean = ops.kv_attention(q, pool.cache, plan)
    assert (clean[starts[2]:starts[3]] == 0).all()
    for which, change, back in ((1, lambda: plan.kv_len[1:2].fill_(16385), lambda: plan.kv_len[1:2].fill_(9000)),
                                (64, lambda: plan.kv_len[64:65].fill_(-1), lambda: plan.kv_len[64:65].fill_(16384)),
                                (3, lambda: plan.page_table[3, 7:8].fill_(-9),
                                 lambda: plan.page_table[3, 7:8].copy_(table[3, 7:8]))):
        keep = plan.page_table.clone()
        change()
        got = ops.kv_attention(q, pool.cache, plan)
        mine = slice(starts[which], starts[which + 1])
        assert got[mine].isnan().all()
        got[mine] = clean[mine]
        plan.page_table.copy_(keep)
        back()
        agree(got, clean, pool, plan, q)  # (lengths move the shares' ends, and with them the order of sums)
    assert torch.equal(ops.kv_attention(q, pool.cache, plan), clean)


def test_the_bound_of_the_many_rows_tests_means_the_tile_form(dev):
    cus = compute_units(dev)
    for rows, heads, group in (([1], 2, 1), ([150, 3], 2, 1), ([4, 1, 1, 4], 2, 7)):
        c = ManyRows(dev, rows, [5000] * len(rows), heads=heads, group=group, seed=1)
        units = len(rows) * heads * -(-c.plan.max_rows * group // 256)
        assert units % cus and cus // (units % cus) >= 2  # some are cut, into as many pieces as fit or 79 // 8
        pieces = min(cus // (units % cus), 79 // 8)
        assert workspace(c.cache, c.plan, c.longer(c.q)) == units % cus * pieces * 256 * 520


@pytest.mark.parametrize("kind,rows", [(Case, [2, 3, 1]), (Case, [20, 5, 4]), (ManyRows, [40, 30, 20])])
def test_rows_that_cannot_be_named_and_rows_beyond_the_bound(dev, kind, rows):
    """More rows than the plan's bound: that many become NaN.  Entries out of order or out of range: left as they are."""
    from diffsynth_engine_amd import kv_cache, ops

    c = kind(dev, rows, [200, 190, 180], page=32, seed=41)
    q = c.longer(c.q) if kind is ManyRows else c.q.to(dev)
    clean = ops.kv_attention(q, c.cache, c.plan)
    s, bound, total = c.starts, c.plan.max_rows, q.shape[0]

    def run(starts):
        plan = kv_cache.KVPlan(c.plan.page_table, torch.tensor(starts, dtype=torch.int32, device=dev), c.plan.kv_len,
                               max_rows=bound, max_kv_len=200)
        out = torch.full_like(q, 7.0)
        return ops.kv_attention(q, c.cache, plan, out=out)

    for starts in ([s[0], s[1], total + 1, s[3]], [s[0], s[1], -2, s[3]], [s[0], s[1], s[1] - 1, s[1] - 1]):
        got = run(starts)
        assert torch.equal(got[:s[1] - 1], clean[:s[1] - 1]) and (got[s[1]:] == 7).all()
    got = run([0, 0, bound + 1, bound + 1])
    assert got[:bound].isnan().all() and (got[bound:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
def test_norm_weights_of_other_types_are_rounded_to_bf16_first(dev, dtype):
    from diffsynth_engine_amd import ops

    w = (1 + 0.2 * torch.randn(128, generator=torch.Generator().manual_seed(2))).to(dtype).to(dev)
    got = []
    for weight in (w, w.bfloat16(), torch.cat((w[:1], w)).bfloat16()[1:]):  # the last: aligned to an element only
        c = Case(dev, [3, 20], [40, 50], group=2, page=16, seed=5)
        out = ops.kv_append(c.k.to(dev), c.v.to(dev), c.cache, c.plan, k_norm_w=weight, q=c.q.to(dev),
                            q_norm_w=weight)
        got.append([out] + [t.view(torch.uint8) for t in (c.cache.k, c.cache.k_scale)])
    assert all(torch.equal(a, b) for x in got[1:] for a, b in zip(got[0], x))


def test_a_prompt_beside_single_rows_is_right_together_and_apart(dev):
    """Slices of one plan's arrays make the plans of two calls."""
    from diffsynth_engine_amd import kv_cache, ops

    pool = Pool(dev, 8, 64, 64, seed=11)
    rows, lens = [700] + [1] * 20, [900] + [3000 - 100 * i for i in range(20)]
    plan, starts, table, q = pool.batch(rows, lens, 4)
    whole = ops.kv_attention(q, pool.cache, plan)
    pool.check(whole, q, starts, table, lens, only=(0, 1, 7, 20))
    for a, b in ((0, 1), (1, 21)):
        first = starts[a]
        part = kv_cache.KVPlan(plan.page_table[a:b], plan.row_start[a:b + 1] - first, plan.kv_len[a:b],
                               max_rows=max(rows[a:b]), max_kv_len=max(lens[a:b]))
        own = slice(first, starts[b])
        got = ops.kv_attention(q[own], pool.cache, part)
        agree(got, whole[own], pool, part, q[own])


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("rows,lens,group,window", [
    ([1], [3000], 4, 500),             # one column
    ([5, 2], [3000, 1700], 7, 333),    # two
    ([40, 9], [3000, 500], 1, 64),
    ([700, 300], [2500, 2000], 20, 900),  # the tile form
    ([1] * 66, [16384 - 7 * i for i in range(66)], 4, 13000),  # even shares
])
def test_pages_in_front_of_every_window_are_not_looked_at(dev, page, rows, lens, group, window):
    """A program with a window gives such pages to others: their table entries may hold anything."""
    from diffsynth_engine_amd import ops

    pool = Pool(dev, 8, 64, page, seed=page + len(rows))
    plan, starts, table, q = pool.batch(rows, lens, group)
    if len(rows) == 66:
        assert workspace(pool.cache, plan, q, window) == 2 * compute_units(dev) * 16 * 520
    clean = ops.kv_attention(q, pool.cache, plan, window=window)
    pool.check(clean, q, starts, table, lens, window=window, only=(0, len(rows) - 1))
    pool.cache.k.view(torch.uint8)[0, :, :, ::5] = 0x7f  # what stands in for a page out of range: NaN here
    pool.cache.v.view(torch.uint8)[0, :, :, ::5] = 0xff
    table = torch.where(table == 0, 1, table)
    plan.page_table.copy_(table)
    clean = ops.kv_attention(q, pool.cache, plan, window=window)
    assert not clean.isnan().any()
    for bad in (-1, 10 ** 9, 0):
        for b, (r, n) in enumerate(zip(rows, lens)):
            plan.page_table[b, :max(n - r + 1 - window, 0) // page] = bad
        assert torch.equal(ops.kv_attention(q, pool.cache, plan, window=window), clean), bad
