"""The paged 8-bit key/value cache on the GPU against its 64-bit oracle.

Tolerances, derived before the first run.
Append: a stored value is the fp32 result rounded to e4m3: half a step, 2^-4 of the value or 2^-10 of the block's scale
among the subnormals.  The fp32 arithmetic before it (sum of 128 squares, root, two products, the rotation's products and
sum) is off by less than 2^-18 of the larger element of the rotated pair.  q: half a bf16 step, 2^-8, beside the same.
Attention, with A = sum_j p_j |v_j|: the bf16 store 2^-8 |o|; fp16 weights 2^-11 A; a score error d moves a weight by
e^d - 1 and the output by at most 2 d A.  d: q's second term leaves 2^-22 of the row's largest element, the matrix
instruction sums 128 products in fp32 (2^-24 of their magnitudes each, 128 of them), and the base-2 argument is rounded
at its magnitude below 2^8 (2^-16): d <= scale * |q|max * sum|k| * 2^-22 + scale * sum|q k| 2^-17 + 2^-15 <= 2^-11 for the
operands here (|q|max < 12, sum |k| < 128, sum |q k| < 500).  Together 2^-8 |o| + 2^-9 A.
"""
import math

import pytest
import torch

from oracle import kv_cache as okv

pytestmark = pytest.mark.gpu

BF, F8, E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
PAGES = (16, 32, 64, 128)


class Case:
    """A cache, a plan and packed rows, on the host (for the oracle) and on the device."""

    def __init__(self, dev, rows, lens, heads=2, group=1, page=64, seed=0, spread=1.0, pad=0, q_scale=1.0, spare=2,
                 max_rows=None, max_kv_len=None):
        from diffsynth_engine_amd import kv_cache

        g = torch.Generator().manual_seed(seed)
        self.rows, self.lens, self.page, self.dev = rows, lens, page, dev
        held = [-(-n // page) for n in lens]
        pool = sum(held) + spare
        order = torch.randperm(pool, generator=g).tolist()
        self.table = []
        for n in held:
            self.table.append(order[:n])
            order = order[n:]
        self.starts = [0]
        for r in rows:
            self.starts.append(self.starts[-1] + r)
        self.total = self.starts[-1] + pad
        self.host = {}
        for n in "kv":
            x = torch.randn(pool, heads, page, 128, generator=g) * 200
            self.host[n] = x.clamp(-448, 448).to(F8)
            e = torch.randn(pool, heads, generator=g) * spread * 3 - 7
            self.host[n + "_scale"] = e.round().to(torch.int32) if n == "v" else torch.full((pool, heads), -7).int()
        self.k, self.v = (torch.randn(self.total, heads, 128, generator=g).bfloat16() for _ in range(2))
        self.q = (q_scale * torch.randn(self.total, heads * group, 128, generator=g)).bfloat16()
        codes = [self.host[n].to(dev) for n in "kv"]
        scales = [(self.host[n + "_scale"] + 127).to(torch.uint8).to(dev).view(E8) for n in "kv"]
        self.cache = kv_cache.KVCache(*codes, *scales)
        width = max(held + [1])
        rows_ = [t + [-1] * (width - len(t)) for t in self.table]
        self.plan = kv_cache.KVPlan(torch.tensor(rows_, dtype=torch.int32, device=dev),
                                    torch.tensor(self.starts, dtype=torch.int32, device=dev),
                                    torch.tensor(lens, dtype=torch.int32, device=dev),
                                    max_rows=max(rows) if max_rows is None else max_rows,
                                    max_kv_len=max(lens) if max_kv_len is None else max_kv_len)
        self.g = g

    def attend(self, q=None, **kw):
        from diffsynth_engine_amd import ops

        return ops.kv_attention(self.q.to(self.dev) if q is None else q, self.cache, self.plan, **kw)

    def want(self, **kw):
        return okv.attention(self.q, self.host, self.table, self.starts, self.lens, **kw)

    def pull(self):
        """The device cache as the oracle takes it."""
        c = self.cache
        return dict(k=c.k.cpu(), v=c.v.cpu(), **{n + "_scale": getattr(c, n + "_scale").view(torch.uint8).cpu().int() - 127
                                                 for n in "kv"})


def close(got, want, size, n):
    got, want, size = got[:n].double().cpu(), want[:n], size[:n]
    assert not got.isnan().any()
    off = (got - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -9 * size)
    assert off.max().item() <= 0, (off.max().item(), off.flatten(1).amax(1).argmax().item())


def check_attend(case, **kw):
    got = case.attend(**kw)
    kw.pop("split_keys", None)
    want, size = case.want(**kw)
    close(got, want, size, case.starts[-1])
    return got


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("kv", [1, 15, 16, 17, 31, 33, 64, 65, 129, 300, 777])
def test_one_token(dev, page, kv):
    check_attend(Case(dev, [1], [kv], page=page, seed=kv))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 7, 33, 200])
@pytest.mark.parametrize("page,group,rows,lens", [
    (64, 1, [1, 3, 2], [100, 3, 260]),
    (16, 7, [5, 1, 2, 4], [333, 2, 64, 4]),
    (128, 4, [9, 4], [129, 500]),
    (32, 1, [40, 17, 70], [50, 300, 70]),
    (64, 2, [130, 1], [400, 31]),
    (16, 1, [300], [300]),
])
def test_ragged_batches(dev, page, group, rows, lens, window, causal):
    check_attend(Case(dev, rows, lens, group=group, page=page, seed=sum(lens)), causal=causal, window=window)


@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_see_nothing_are_zero(dev, causal):
    # more rows than tokens, no tokens at all, and no rows
    c = Case(dev, [6, 3, 0, 40, 2], [4, 0, 20, 7, 9], page=16, group=3, seed=3)
    got = check_attend(c, causal=causal)
    nothing = [6, 7, 8] + ([0, 1] + list(range(9, 42)) if causal else [])
    assert (got[nothing] == 0).all()


@pytest.mark.parametrize("rows,lens,group", [([1] * 3, [2000, 900, 1], 4), ([3, 2], [1999, 40], 5), ([25], [1200], 1),
                                             ([70], [1500], 1), ([150, 3], [700, 1000], 2)])
def test_split_and_unsplit_agree_with_the_oracle_and_repeat_their_bits(dev, rows, lens, group):
    c = Case(dev, rows, lens, group=group, seed=9)
    a = check_attend(c)
    b = check_attend(c, split_keys=False)
    assert torch.equal(a, c.attend()) and torch.equal(b, c.attend(split_keys=False))


def test_scales_far_apart_and_peaked_scores(dev):
    # block exponents of V over forty powers of two: each block's weight must not be lost beside the others'
    check_attend(Case(dev, [1, 2], [500, 900], page=16, spread=3.0, seed=12))
    c = Case(dev, [2, 20], [700, 300], page=32, q_scale=2.0, seed=13)
    check_attend(c, scale=0.5 / math.sqrt(128))
    c.host["v_scale"][::2], c.host["v_scale"][1::2] = -48, 48
    c.cache.v_scale.view(torch.uint8).copy_((c.host["v_scale"] + 127).to(torch.uint8))
    check_attend(c)


def test_strided_rows_and_rows_behind_the_last_sequence(dev):
    c = Case(dev, [3, 5], [70, 90], group=2, pad=4, seed=21)
    want, size = c.want()
    wide = torch.zeros(c.total, 9, 136, dtype=BF, device=dev)
    q = wide[:, 2:6, :128]
    q.copy_(c.q)
    buf = torch.full((c.total, 6, 128), 7.0, dtype=BF, device=dev)
    out = buf.transpose(0, 1).contiguous().transpose(0, 1)[:, 1:5]  # head-major
    out.fill_(7.0)
    assert c.attend(q=q, out=out) is out
    close(out, want, size, 8)
    assert (out[8:] == 7).all()


def test_nan_where_rows_do_not_look_stays_there(dev):
    """Codes behind a sequence's end, of masked tokens and before a window: NaN in K and V reaches only rows that see
    it."""
    for page, rows, window in ((16, 5, 0), (64, 5, 20), (64, 40, 0), (64, 140, 30), (128, 2, 0)):
        n = 150
        c = Case(dev, [rows], [n], page=page, seed=page)
        clean = c.attend(window=window)
        for t in c.table[0][-1:]:
            for code in (c.cache.k, c.cache.v):
                tail = code.view(torch.uint8)[t, :, n % page:]
                if n % page:
                    tail.fill_(0x7f)
        assert torch.equal(c.attend(window=window), clean)
        for token in (n - 1, n - rows + 1, 3):  # seen by the rows from it on, as long as the window lasts
            at, off = c.table[0][token // page], token % page
            for code, which in ((c.cache.v, "v"), (c.cache.k, "k")):
                raw = code.view(torch.uint8)
                old = raw[at, 0, off, 5].clone()
                raw[at, 0, off, 5] = 0xff
                got = c.attend(window=window)
                pos = torch.arange(n - rows, n)
                sees = (pos >= token) & ((pos < token + window) if window else torch.ones_like(pos, dtype=torch.bool))
                sees = sees.to(dev)
                if which == "v":
                    assert got[sees, 0, 5].isnan().all()
                    got = got.clone()
                    got[sees, 0, 5] = clean[sees, 0, 5]
                else:
                    assert got[sees, 0].isnan().all()
                    got = got.clone()
                    got[sees, 0] = clean[sees, 0]
                assert torch.equal(got, clean), (page, rows, window, token, which)
                raw[at, 0, off, 5] = old


def test_nan_and_infinite_queries_and_scales(dev):
    c = Case(dev, [3, 30], [90, 80], seed=31)
    clean = c.attend()
    q = c.q.to(dev)
    q[1, 0, 7] = math.nan
    q[12, 1, 100] = math.inf
    got = c.attend(q=q)
    assert got[1, 0].isnan().all() and got[12, 1].isnan().all()
    got[1, 0], got[12, 1] = clean[1, 0], clean[12, 1]
    assert torch.equal(got, clean)
    c.cache.v_scale.view(torch.uint8)[c.table[0][0], 1] = 255
    got = c.attend()
    assert got[:3, 1].isnan().all() and not got[:3, 0].isnan().any() and torch.equal(got[3:], clean[3:])


def test_bad_metadata_is_contained(dev):
    """Page numbers and lengths out of range become NaN rows or rows left alone, and no other row changes."""
    for rows in ([2, 3, 1], [40, 30, 20], [150, 10, 20]):
        c = Case(dev, rows, [200, 190, 180], page=32, seed=41)
        clean, s = c.attend(), c.starts
        for bad in (-5, 10 ** 9):
            keep = c.plan.page_table[1, 2].clone()
            c.plan.page_table[1, 2] = bad
            got = c.attend()
            assert got[s[1]:s[2]].isnan().all()
            assert torch.equal(got[:s[1]], clean[:s[1]]) and torch.equal(got[s[2]:], clean[s[2]:])
            c.plan.page_table[1, 2] = keep
        for bad in (-1, 201, 2 ** 31 - 1):
            c.plan.kv_len[1] = bad
            got = c.attend()
            assert got[s[1]:s[2]].isnan().all()
            assert torch.equal(got[:s[1]], clean[:s[1]]) and torch.equal(got[s[2]:], clean[s[2]:])
        c.plan.kv_len[1] = 190
        for at, bad in ((2, s[1] - 1), (2, -3), (2, c.total + 1)):  # rows that cannot be named: the neighbours' too
            c.plan.row_start[at] = bad
            out = torch.full_like(clean, 7.0)
            got = c.attend(out=out)
            own = min(s[1], bad) if bad >= 0 else s[1]  # rows that sequence 0 shares with nobody
            assert torch.equal(got[:own], clean[:own])
            assert (got[s[2]:] == 7).all() or bad == s[1] - 1
            c.plan.row_start[at] = s[2]
        assert torch.equal(c.attend(), clean)


def test_offsets_beyond_32_bits(dev):
    from diffsynth_engine_amd import kv_cache, ops

    pages, page = 70000, 64
    raw = torch.zeros(pages * 9 * page * 128, dtype=torch.uint8, device=dev)  # 5.2 GB: pages nine blocks apart
    view = raw.view(pages, 9, page, 128)
    c = Case(dev, [2], [130], heads=1, seed=51)
    far = [pages - 1, 7, pages - 30000]
    k, v = view[:, 3:4].view(F8), view[:, 8:9].view(F8)
    scales = [torch.full((pages, 1), 127, dtype=torch.uint8, device=dev).view(E8) for _ in range(2)]
    for i, p in enumerate(c.table[0]):
        for big, small, n in ((k, c.cache.k, 0), (v, c.cache.v, 1)):
            big.view(torch.uint8)[far[i]] = small.view(torch.uint8)[p]
            scales[n].view(torch.uint8)[far[i]] = (c.cache.k_scale, c.cache.v_scale)[n].view(torch.uint8)[p]
    cache = kv_cache.KVCache(k, v, *scales)
    plan = kv_cache.KVPlan(torch.tensor([far], dtype=torch.int32, device=dev), c.plan.row_start, c.plan.kv_len,
                           max_rows=2, max_kv_len=130)
    assert torch.equal(ops.kv_attention(c.q.to(dev), cache, plan), c.attend())
    x = c.k.to(dev)
    ops.kv_append(x, x, cache, plan)
    ops.kv_append(x, x, c.cache, c.plan)
    for i, p in enumerate(c.table[0]):
        assert torch.equal(k.view(torch.uint8)[far[i]], c.cache.k.view(torch.uint8)[p])
        assert torch.equal(v.view(torch.uint8)[far[i]], c.cache.v.view(torch.uint8)[p])


# ------------------------------------------------------------------------------------------------ append

def rope_rows(batch, rows, seed=0):
    ang = torch.rand(batch, rows, 64, generator=torch.Generator().manual_seed(seed)) * 6.28
    return torch.stack((ang.cos(), ang.sin()), -1)


def run_append(case, **kw):
    from diffsynth_engine_amd import ops

    kw = {n: t.to(case.dev) if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    return ops.kv_append(case.k.to(case.dev), case.v.to(case.dev), case.cache, case.plan, **kw)


def check_append(case, q=None, q_norm_w=None, **kw):
    before = case.pull()
    want = okv.append(before, case.table, case.starts, case.lens, case.k, case.v, **kw)
    got_q = run_append(case, q=q, q_norm_w=q_norm_w, **kw)
    after = case.pull()
    touched = set()
    for b, (r, n) in enumerate(zip(case.rows, case.lens)):
        touched |= set(case.table[b][(n - r) // case.page:-(-n // case.page)] if r else ())
    big = 1.0 if kw.get("rope") is None else None
    for name in "kv":
        exact, exps = want[name]
        assert torch.equal(after[name + "_scale"], exps), name
        got = okv.values(after[name], torch.zeros_like(exps))
        noise = 2.0 ** -18 * exact.abs()
        if name == "k" and big is None:
            noise = 2.0 ** -18 * exact.unflatten(-1, (64, 2)).abs().amax(-1, keepdim=True).expand(
                *exact.shape[:-1], 64, 2).flatten(-2)
        ok = (got - exact).abs() <= torch.maximum(2.0 ** -4 * exact.abs(), torch.tensor(2.0 ** -10)) * (1 + 2.0 ** -10) + noise
        ok |= got.isnan() & exact.isnan()
        assert ok.all(), name
        rest = [p for p in range(case.cache.pages) if p not in touched]
        assert torch.equal(after[name].view(torch.uint8)[rest], before[name].view(torch.uint8)[rest])
    for b, (r, n) in enumerate(zip(case.rows, case.lens)):  # tokens behind the appended ones are left alone
        if r and n % case.page:
            p = case.table[b][-1]
            for name in "kv":
                a, z = (t[name].view(torch.uint8)[p, :, n % case.page:] for t in (after, before))
                assert torch.equal(a, z)
    if q is not None:
        rope = kw.get("rope")
        for b, (r, n) in enumerate(zip(case.rows, case.lens)):
            part = slice(case.starts[b], case.starts[b + 1])
            table = None if rope is None else rope[b if rope.shape[0] > 1 else 0]
            exact = okv.norm_rope(q[part], q_norm_w, table, torch.arange(n - r, n))
            pair = exact.unflatten(-1, (64, 2)).abs().amax(-1, keepdim=True).expand(*exact.shape[:-1], 64, 2).flatten(-2)
            assert ((got_q[part].cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -18 * pair).all()
    return got_q


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("rows,lens", [([1], [1]), ([1, 1], [16, 17]), ([1, 1, 1], [128, 129, 65]), ([3, 0, 20], [40, 9, 20]),
                                       ([130, 7], [200, 500]), ([64], [64])])
@pytest.mark.parametrize("norm,rope", [(False, 0), (True, 1), (True, 0), (False, 3)])
def test_append(dev, page, rows, lens, norm, rope):
    c = Case(dev, rows, lens, heads=3, group=2, page=page, seed=sum(rows) + page)
    w = lambda: (1 + 0.2 * torch.randn(128, generator=c.g)).bfloat16()  # noqa: E731
    kw = dict(k_norm_w=w() if norm else None)
    if rope:
        kw["rope"] = rope_rows(1 if rope == 1 else len(rows), max(lens) + 2)
    check_append(c, q=c.q, q_norm_w=w() if norm else None, **kw)


def test_append_one_at_a_time_moves_the_scale_up_and_never_down(dev):
    from diffsynth_engine_amd import ops

    page, n = 16, 40
    c = Case(dev, [1], [n], heads=2, page=page, seed=61)
    size = torch.tensor([1.0, 0.01, 3.0, 100.0, 2.0, 0.5, 1e4, 1.0])
    held = dict(c.host)
    for t in range(n):
        x = (c.k[:1].float().roll(t, -1) * size[t % 8]).bfloat16()
        y = (c.v[:1].float().roll(3 * t, -1) * size[(t + 3) % 8]).bfloat16()
        c.plan.kv_len.fill_(t + 1)
        want = okv.append(held, c.table, [0, 1], [t + 1], x, y)
        for again in range(2):  # the same row once more changes nothing
            ops.kv_append(x.to(dev), y.to(dev), c.cache, c.plan)
            after = c.pull()
            for name in "kv":
                exact, exps = want[name]
                assert torch.equal(after[name + "_scale"], exps)
                assert torch.equal(okv.values(after[name], torch.zeros_like(exps)), okv.e4m3_nearest(exact)), (t, name)
        held = after


def test_append_special_values(dev):
    c = Case(dev, [20], [20], heads=1, page=32, seed=71)
    c.k[3, 0, 4], c.k[5, 0, 6], c.k[7, 0, 8] = math.inf, -math.inf, math.nan
    c.v[:] = 0
    check_append(c)
    at = c.table[0][0]
    got = c.pull()
    assert got["k"][at, 0, 3, 4].float() == 448 and got["k"][at, 0, 5, 6].float() == -448
    assert got["k"][at, 0, 7, 8].float().isnan() and got["v_scale"][at, 0] == -48 and (got["v"][at, 0, :20].float() == 0).all()
    c.k[:], c.v[:] = 1e30, -1e-30  # beyond both ends of the scales
    check_append(c)
    # the largest finite magnitude sits on both sides of 448 * 2^e
    for x, e in ((448.0, 0), (450.0, 1), (1.75, -8), (1.7578125, -7)):
        c.k[:], c.v[:] = 0.001, 0.001
        c.k[2, 0, 100] = x
        check_append(c)
        assert c.pull()["k_scale"][at, 0] == e


def test_append_prepares_q_in_place_and_from_one_projection(dev):
    from diffsynth_engine_amd import ops

    c = Case(dev, [4, 3], [30, 50], heads=2, group=3, page=16, pad=2, seed=81)
    packed = torch.cat((c.q, c.k, c.v), 1).to(dev)
    w = (1 + 0.2 * torch.randn(128, generator=c.g)).bfloat16().to(dev)
    rope = rope_rows(1, 50).to(dev)
    apart = ops.kv_append(c.k.to(dev), c.v.to(dev), c.cache, c.plan, k_norm_w=w, rope=rope, q=c.q.to(dev), q_norm_w=w)
    first = c.pull()
    q, k, v = packed[:, :6], packed[:, 6:8], packed[:, 8:]
    tail = packed[7:].clone()
    assert ops.kv_append(k, v, c.cache, c.plan, k_norm_w=w, rope=rope, q=q, q_norm_w=w, q_out=q) is q
    assert torch.equal(q[:7], apart[:7]) and torch.equal(packed[7:], tail)
    second = c.pull()
    assert all(torch.equal(first[n].view(torch.uint8) if n in "kv" else first[n],
                           second[n].view(torch.uint8) if n in "kv" else second[n]) for n in first)


def test_append_leaves_out_what_breaks_a_bound(dev):
    for change in (lambda p: p.kv_len[1:2].fill_(2), lambda p: p.kv_len[1:2].fill_(10 ** 9),
                   lambda p: p.kv_len[1:2].fill_(-4), lambda p: p.page_table[1, :2].fill_(-1),
                   lambda p: p.page_table[1, :2].fill_(2 ** 31 - 1), lambda p: p.row_start[1:].fill_(10 ** 6)):
        c = Case(dev, [2, 5, 3], [20, 20, 20], page=16, seed=91)
        before = c.pull()
        change(c.plan)
        run_append(c)
        after = c.pull()
        for p in c.table[1]:
            for n in "kv":
                assert torch.equal(after[n].view(torch.uint8)[p], before[n].view(torch.uint8)[p])
                assert torch.equal(after[n + "_scale"][p], before[n + "_scale"][p])


# ------------------------------------------------------------------------------------------------ together

def test_a_prompt_then_single_tokens_then_a_chunk(dev):
    """The cache as a program uses it: a ragged prompt, single tokens, a few at a time; outputs against the oracle on
    what the cache then holds, and on the unquantised values within e4m3's share."""
    from diffsynth_engine_amd import kv_cache, ops

    g = torch.Generator().manual_seed(7)
    heads, group, page, B = 2, 4, 32, 3
    cache = kv_cache.KVCache.empty(40, heads, page, dev)
    table = torch.randperm(40, generator=g)[:36].view(B, 12).to(torch.int32)
    plan = kv_cache.KVPlan(table.to(dev), torch.zeros(B + 1, dtype=torch.int32, device=dev),
                           torch.zeros(B, dtype=torch.int32, device=dev), max_rows=100, max_kv_len=384)
    w = (1 + 0.2 * torch.randn(128, generator=g)).bfloat16()
    rope = rope_rows(1, 384)
    lens = [0] * B
    hist = [[], [], []]
    for rows in ([100, 31, 64], [1, 1, 1], [1, 1, 1], [1, 0, 1], [5, 3, 17], [1, 1, 1]):
        starts = [0, rows[0], rows[0] + rows[1], sum(rows)]
        lens = [a + b for a, b in zip(lens, rows)]
        plan.row_start.copy_(torch.tensor(starts, dtype=torch.int32))
        plan.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        qkv = torch.randn(sum(rows), heads * (group + 2), 128, generator=g).bfloat16()
        d = qkv.to(dev)
        q, k, v = d[:, :heads * group], d[:, heads * group:-heads], d[:, -heads:]
        plan.check(cache, sum(rows))
        q2 = ops.kv_append(k, v, cache, plan, k_norm_w=w.to(dev), rope=rope.to(dev), q=q, q_norm_w=w.to(dev))
        got = ops.kv_attention(q2, cache, plan)
        held = dict(k=cache.k.cpu(), v=cache.v.cpu(), k_scale=cache.k_scale.view(torch.uint8).cpu().int() - 127,
                    v_scale=cache.v_scale.view(torch.uint8).cpu().int() - 127)
        want, size = okv.attention(q2.cpu(), held, table.tolist(), starts, lens)
        close(got, want, size, sum(rows))
        for b in range(B):
            part = slice(starts[b], starts[b + 1])
            pos = torch.arange(lens[b] - rows[b], lens[b])
            hist[b].append((okv.norm_rope(qkv[part, heads * group:-heads], w, rope[0], pos), qkv[part, -heads:].double()))
            kk, vv = (torch.cat([x[i] for x in hist[b]]) for i in range(2))
            qq = okv.norm_rope(qkv[part, :heads * group], w, rope[0], pos)
            for h in range(heads * group):
                s = qq[:, h] @ kk[:, h // group].T / math.sqrt(128)
                s = s.masked_fill(torch.arange(lens[b])[None] > pos[:, None], -math.inf)
                ref = torch.softmax(s, -1) @ vv[:, h // group]
                err = (got[part, h].double().cpu() - ref).norm() / ref.norm() if rows[b] else torch.tensor(0.0)
                assert err < 2.0 ** -4  # each stored value is within 2^-4; errors of many tokens average below that


def test_another_stream_and_graph_replays(dev):
    """Captured once, replayed with other rows and lengths between eager work; every replay against the eager call."""
    from diffsynth_engine_amd import kv_cache, ops

    g = torch.Generator().manual_seed(17)
    heads, group, page, B, most = 2, 4, 64, 4, 1600
    cache = kv_cache.KVCache.empty(110, heads, page, dev)
    twin = kv_cache.KVCache.empty(110, heads, page, dev)
    for c in (cache, twin):
        for n in "kv":
            codes = (torch.randn(110, heads, page, 128, generator=torch.Generator().manual_seed(1)) * 100).clamp(-448, 448)
            getattr(c, n).copy_(codes.to(F8))
            getattr(c, n + "_scale").view(torch.uint8).fill_(121)
    table = torch.randperm(110, generator=g)[:B * 25].view(B, 25).to(torch.int32).to(dev)
    starts = torch.arange(B + 1, dtype=torch.int32, device=dev)
    lens = torch.tensor([1, 700, 1500, 64], dtype=torch.int32, device=dev)
    plan = kv_cache.KVPlan(table, starts, lens, max_rows=1, max_kv_len=most)
    rope = rope_rows(1, most).to(dev)
    x = torch.randn(B, heads * (group + 2), 128, generator=g).bfloat16().to(dev)

    def step(c):
        q = ops.kv_append(x[:, heads * group:-heads], x[:, -heads:], c, plan, rope=rope, q=x[:, :heads * group])
        return ops.kv_attention(q, c, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(cache)
        first.record_stream(torch.cuda.current_stream())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, step(twin))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(6):
        x.copy_(torch.randn(x.shape, generator=g).bfloat16())
        lens.add_(1)
        eager = step(twin)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, eager), i
        assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8))
        assert torch.equal(cache.v_scale.view(torch.uint8), twin.v_scale.view(torch.uint8))
        (torch.randn(256, 256, device=dev) @ torch.randn(256, 256, device=dev)).sum().item()


def test_two_streams_at_once(dev):
    c, d = Case(dev, [1, 1], [1500, 800], group=4, seed=1), Case(dev, [2], [1900], heads=4, seed=2)
    a, b = c.attend(), d.attend()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    qa, qb = c.q.to(dev), d.q.to(dev)
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(one):
            x = c.attend(q=qa)
        with torch.cuda.stream(two):
            y = d.attend(q=qb)
        torch.cuda.synchronize()
        assert torch.equal(x, a) and torch.equal(y, b)


def test_refusals(dev):
    from diffsynth_engine_amd import kv_cache, ops

    c = Case(dev, [2, 3], [40, 50], group=2, page=16, seed=5)
    q, k, v = c.q.to(dev), c.k.to(dev), c.v.to(dev)
    w, rope = torch.ones(128, dtype=BF, device=dev), rope_rows(1, 50).to(dev)
    for kw in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :64]), dict(q=q[0]), dict(q=q.transpose(1, 2)),
               dict(window=-1), dict(scale=0.0), dict(scale=math.inf), dict(scale=-1.0), dict(scale=math.nan),
               dict(out=torch.empty_like(q[:4])), dict(out=torch.empty_like(q, dtype=torch.float16)),
               dict(out=torch.empty_like(q[:, :2])), dict(q=torch.zeros(5, 4, 130, dtype=BF, device=dev)[..., 1:129])):
        args = dict(q=q)
        args.update(kw)
        with pytest.raises(ValueError):
            ops.kv_attention(args.pop("q"), c.cache, c.plan, **args)
    for kw in (dict(k=k[:, :1]), dict(v=v[:4]), dict(k=k.float()), dict(k_norm_w=w[:64]), dict(q_norm_w=w),
               dict(q_out=torch.empty_like(q)), dict(q=q[:4]), dict(q=q, q_out=q[:, :2]), dict(eps=-1.0),
               dict(rope=rope[:, :49]), dict(rope=rope.double()), dict(rope=rope.expand(3, -1, -1, -1))):
        args = dict(k=k, v=v)
        args.update(kw)
        with pytest.raises(ValueError):
            ops.kv_append(args.pop("k"), args.pop("v"), c.cache, c.plan, **args)
    for host in (dict(k=c.k), dict(rope=rope.cpu()), dict(q=c.q), dict(k_norm_w=w.cpu())):
        args = dict(k=k, v=v)
        args.update(host)
        with pytest.raises(RuntimeError):
            ops.kv_append(args.pop("k"), args.pop("v"), c.cache, c.plan, **args)
    far = kv_cache.KVCache.empty(2, 2, 16, "cpu")
    with pytest.raises(ValueError):
        ops.kv_attention(q, far, c.plan)
    none = q[:0]
    assert ops.kv_attention(none, c.cache, c.plan).shape == none.shape
    assert ops.kv_append(k[:0], v[:0], c.cache, c.plan) is None


class Pool:
    """Random pages that the page tables of many sequences share, and the same formulas in 64 bits on the device."""

    def __init__(self, dev, heads, pages, page, seed=0):
        from diffsynth_engine_amd import kv_cache

        self.dev, self.page, self.heads, self.g = dev, page, heads, torch.Generator(dev).manual_seed(seed)
        put = lambda scale: (torch.randn(pages, heads, page, 128, generator=self.g, device=dev) * scale).clamp(-448, 448).to(F8)
        self.codes = put(128.0), put(200.0)  # times 2^-7 below: keys of deviation 1
        v_exp = torch.randint(-12, 1, (pages, heads), generator=self.g, device=dev)
        self.exps = torch.full_like(v_exp, -7), v_exp
        self.cache = kv_cache.KVCache(*self.codes, *[(e + 127).to(torch.uint8).view(E8) for e in self.exps])

    def batch(self, rows, lens, group):
        """(plan, starts, table, q)"""
        from diffsynth_engine_amd import kv_cache

        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        width = -(-max(lens) // self.page)
        table = torch.randint(0, self.codes[0].shape[0], (len(rows), width), generator=self.g, device=self.dev).int()
        q = torch.randn(starts[-1], self.heads * group, 128, generator=self.g, device=self.dev).bfloat16()
        return kv_cache.KVPlan(table, ints(starts), ints(lens), max_rows=max(rows), max_kv_len=max(lens)), starts, table, q

    def value(self, i, pages, n):
        """(heads, n, 128) fp64 of the first n tokens on these pages"""
        held = pages[: -(-n // self.page)].long()
        x = self.codes[i][held].double() * torch.exp2(self.exps[i][held].double())[..., None, None]
        return x.transpose(0, 1).flatten(1, 2)[:, :n].contiguous()

    def check(self, out, q, starts, table, lens, causal=True, window=0, only=None):
        group = q.shape[1] // self.heads
        for b in range(len(lens)) if only is None else only:
            r, n = starts[b + 1] - starts[b], lens[b]
            if r == 0:
                continue
            got = out[starts[b]:starts[b + 1]].double()
            if n == 0:
                assert (got == 0).all()
                continue
            k, v = self.value(0, table[b], n), self.value(1, table[b], n)
            end = torch.arange(n - r + 1, n + 1, device=self.dev) if causal else torch.full((r,), n, device=self.dev)
            pos = torch.arange(n, device=self.dev)
            see = pos < end[:, None]
            if window:
                see &= pos >= end[:, None] - window
            for h in range(self.heads):
                x = q[starts[b]:starts[b + 1], h * group:(h + 1) * group].double().transpose(0, 1).flatten(0, 1)
                s = x @ k[h].t().contiguous() / math.sqrt(128)
                p = torch.softmax(s.masked_fill(~see.repeat(group, 1), -math.inf), -1)
                p = torch.where(see.repeat(group, 1), p, 0.0)  # rows that see nothing
                want, size = (p @ v[h]).view(group, r, 128), (p @ v[h].abs()).view(group, r, 128)
                off = (got[:, h * group:(h + 1) * group].transpose(0, 1) - want).abs()
                assert (off - (2.0 ** -8 * want.abs() + 2.0 ** -9 * size)).max().item() <= 0, (b, h)


@pytest.mark.parametrize("batch,heads,group,top,most_rows", [
    (70, 8, 4, 16384, 3),     # long ragged caches
    (700, 8, 1, 1700, 1),     # many sequences
    (66, 32, 5, 4097, 3),     # two units meet in one share
    (1, 40, 1, 150000, 1),    # few units: every share is a piece of one
])
def test_even_shares_of_long_caches(dev, batch, heads, group, top, most_rows):
    # more than 512 tiles of 32 tokens for every compute unit, by the plan's own bounds
    from diffsynth_engine_amd import ops

    g = torch.Generator().manual_seed(batch)
    pool = Pool(dev, heads, 64, 64, seed=batch)
    lens = torch.randint(0, top + 1, (batch,), generator=g).tolist()
    lens[0] = top
    rows = [min(int(r), n) if i % 5 else 1 for i, (r, n) in enumerate(zip(torch.randint(0, most_rows + 1, (batch,), generator=g),
                                                                          lens))]
    plan, starts, table, q = pool.batch(rows, lens, group)
    cus = torch.cuda.get_device_properties(dev).multi_processor_count
    if batch > 1:
        assert batch * heads * (top // 32 + 1) >= 512 * cus
    for kw in (dict(), dict(window=1000), dict(causal=False)):
        out = ops.kv_attention(q, pool.cache, plan, **kw)
        pool.check(out, q, starts, table, lens, only=None if batch <= 70 and not kw else range(0, batch, 13), **kw)
        assert torch.equal(out, ops.kv_attention(q, pool.cache, plan, **kw))


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("rows,lens,heads,group,kw", [
    ([300, 257], [9001, 4200], 1, 1, {}),                       # tile form, page numbers loaded more than once
    ([300], [9001], 1, 1, dict(causal=False, split_keys=False)),
    ([3, 1], [40001, 16500], 2, 2, dict(split_keys=False)),     # streaming form, the same
    ([8], [20000], 2, 4, dict(window=17000, split_keys=False)),
    ([9, 5], [3000, 700], 4, 7, {}),                            # two blocks of two columns
    ([60], [2000], 3, 1, {}),
    ([33, 1], [1000, 2000], 2, 1, dict(causal=False)),
    ([900], [1700], 5, 20, {}),                                 # units behind the last whole round are cut
    ([900], [1700], 5, 20, dict(causal=False, window=1200)),
])
def test_long_key_ranges_and_forms_in_between(dev, page, rows, lens, heads, group, kw):
    from diffsynth_engine_amd import ops

    pool = Pool(dev, heads, 100, page, seed=page)
    plan, starts, table, q = pool.batch(rows, lens, group)
    out = ops.kv_attention(q, pool.cache, plan, **kw)
    kw = {n: x for n, x in kw.items() if n != "split_keys"}
    pool.check(out, q, starts, table, lens, **kw)


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("rows", [1, 20, 50, 300])
@pytest.mark.parametrize("shape", ["rise", "fall", "spike", "late"])
def test_scores_that_move_the_reference(dev, page, rows, shape):
    # Scores up to |q| |k| = 128 * 6 / sqrt(128) = 68 for the row that agrees with u.  The terms of the bound above:
    # scale |q|max sum|k| 2^-22 = 0.09 * 5 * 900 * 2^-22 < 2^-13, scale sum|q k| 2^-17 < 85 * 2^-17 < 2^-10.5 and 2^-15:
    # 2 d + 2^-11 < 2^-9.4 + 2^-11 + 2^-11.4 < 2^-8.5; the third term of `close` is taken twice for it.
    c = Case(dev, [rows], [max(rows, 1) + 1500], page=page, seed=rows)
    n, g = c.lens[0], c.g
    u = torch.randn(128, generator=g).sign()
    t = torch.arange(n, dtype=torch.float32)
    height = {"rise": 6 * t / n, "fall": 6 - 6 * t / n, "spike": 6.0 * (t == 700), "late": 6.0 * (t >= n - rows - 40)}[shape]
    k = height[:, None, None] * u + 0.25 * torch.randn(n, 2, 128, generator=g)
    for p, at in enumerate(c.table[0]):
        x = k[p * page:(p + 1) * page] * 16  # e4m3's normal numbers: exponent -4 below
        c.host["k"][at, :, :x.shape[0]] = x.transpose(0, 1).to(F8)
    c.host["k_scale"].fill_(-4)
    c.cache.k.copy_(c.host["k"].to(dev))
    c.cache.k_scale.view(torch.uint8).fill_(123)
    sign = torch.tensor([1.0, -1.0, 0.1])[torch.arange(c.total) % 3]
    c.q = (sign[:, None, None] * u + 0.05 * torch.randn(c.total, 2, 128, generator=g)).bfloat16()
    for causal in (True, False):
        got = c.attend(causal=causal)
        want, size = c.want(causal=causal)
        close(got, want, 2 * size, c.starts[-1])


@pytest.mark.parametrize("rows,lens,window", [([5], [200], 0), ([40], [200], 0), ([150, 3], [200, 150], 40), ([3] * 4, [2000] * 4, 0)])
def test_a_scale_of_nan_reaches_only_rows_that_see_its_block(dev, rows, lens, window):
    for page in (16, 64):
        c = Case(dev, rows, lens, group=2, page=page, seed=page)
        clean = c.attend(window=window)
        for at in (lens[0] - 2, lens[0] - rows[0]):  # the block of this token
            for scale in (c.cache.k_scale, c.cache.v_scale):
                raw = scale.view(torch.uint8)
                old = raw[c.table[0][at // page], 1].clone()
                raw[c.table[0][at // page], 1] = 255
                got = c.attend(window=window)
                raw[c.table[0][at // page], 1] = old
                first, last = at // page * page, min(at // page * page + page, lens[0]) - 1  # the block's tokens
                pos = torch.arange(lens[0] - rows[0], lens[0])
                sees = (pos >= first) & ((pos - window < last) if window else torch.ones_like(pos, dtype=torch.bool))
                mine = torch.zeros(c.total, 4, dtype=torch.bool)
                mine[:rows[0], 2:] = sees[:, None]
                mine = mine.to(dev)
                assert got[mine].isnan().all() and torch.equal(got[~mine], clean[~mine]), (page, at)


def test_no_tokens_at_all(dev):
    for rows in ([1, 2], [20, 3], [300, 1]):
        c = Case(dev, rows, [0, 0], group=2, seed=1)
        for bound in (0, 4096):
            from diffsynth_engine_amd import kv_cache

            plan = kv_cache.KVPlan(torch.zeros(2, 64, dtype=torch.int32, device=dev), c.plan.row_start, c.plan.kv_len,
                                   max_rows=max(rows), max_kv_len=bound)
            c.plan = plan
            assert (c.attend() == 0).all() and (c.attend(causal=False, window=3) == 0).all()


@pytest.mark.parametrize("rows,lens", [([1, 3], [3000, 50]), ([30], [700]), ([600], [900])])
def test_out_may_be_q(dev, rows, lens):
    c = Case(dev, rows, lens, group=3, seed=rows[0])
    q, want = c.q.to(dev), c.attend()
    assert c.attend(q=q, out=q) is q and torch.equal(q, want)


def test_outputs_that_overlap_are_refused(dev):
    from diffsynth_engine_amd import ops

    c = Case(dev, [2, 3], [40, 50], group=2, page=16, seed=5)
    q, k, v = c.q.to(dev), c.k.to(dev), c.v.to(dev)
    flat = torch.empty(5 * 9 * 128, dtype=BF, device=dev)
    for bad in (q[:1].expand(5, -1, -1), q[:, :1].expand(-1, 4, -1), flat.as_strided((5, 4, 128), (256, 128, 1))):
        with pytest.raises(ValueError):
            ops.kv_attention(q, c.cache, c.plan, out=bad)
        with pytest.raises(ValueError):
            ops.kv_append(k, v, c.cache, c.plan, q=q, q_out=bad)
    out = flat.view(5, 9, 128)[:, 1:8:2]  # every other head of a wider buffer
    assert torch.equal(ops.kv_attention(q, c.cache, c.plan, out=out), ops.kv_attention(q, c.cache, c.plan))


def test_a_q_without_heads_does_not_keep_k_and_v_out(dev):
    from diffsynth_engine_amd import ops

    c, d = (Case(dev, [3, 1], [20, 40], page=16, seed=7) for _ in range(2))
    q = torch.empty(4, 0, 128, dtype=BF, device=dev)
    assert ops.kv_append(c.k.to(dev), c.v.to(dev), c.cache, c.plan, q=q).shape == q.shape
    ops.kv_append(d.k.to(dev), d.v.to(dev), d.cache, d.plan)
    a, b = c.pull(), d.pull()
    assert all(torch.equal(a[n].view(torch.uint8), b[n].view(torch.uint8)) and torch.equal(a[n + "_scale"], b[n + "_scale"])
               for n in "kv")
    assert not torch.equal(a["k"].view(torch.uint8), c.host["k"].view(torch.uint8))


# ------------------------------------------------------------------------------------------------ the form for many rows

class ManyRows(Case):
    """The same batch under a bound on its rows that sends it to the form for many of them, with as many rows behind it."""

    def __init__(self, dev, rows, lens, heads=2, group=1, **kw):
        bound = 32 * 260 // (group * heads * len(rows)) + 64  # more blocks of 32 rows than compute units
        kw["max_rows"] = max(bound, *rows)
        super().__init__(dev, rows, lens, heads=heads, group=group, **kw)

    def longer(self, q):
        q = q.to(self.dev)
        return torch.cat((q, torch.full((self.plan.max_rows, *q.shape[1:]), math.nan, dtype=BF, device=self.dev)))

    def attend(self, q=None, **kw):
        q = self.longer(self.q if q is None else q)
        out = torch.full(q.shape, 7.0, dtype=BF, device=self.dev)
        assert super().attend(q=q, out=out, **kw) is out
        assert (out[self.total:] == 7).all()
        return out[:self.total]


@pytest.fixture
def many_rows(monkeypatch):
    monkeypatch.setitem(globals(), "Case", ManyRows)


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("kv", [1, 16, 63, 64, 65, 129, 777])
def test_many_rows_one_token(dev, many_rows, page, kv):
    check_attend(Case(dev, [1], [kv], page=page, seed=kv))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 33, 200])
@pytest.mark.parametrize("page,group,rows,lens", [
    (64, 1, [1, 3, 2], [100, 3, 260]),
    (16, 7, [5, 1, 2, 4], [333, 2, 64, 4]),
    (128, 4, [9, 4], [129, 500]),
    (32, 1, [40, 17, 70], [50, 300, 70]),
    (64, 2, [130, 1], [400, 31]),
    (16, 1, [300], [300]),
    (64, 3, [260], [520]),
])
def test_many_rows_ragged(dev, many_rows, page, group, rows, lens, window, causal):
    check_attend(Case(dev, rows, lens, group=group, page=page, seed=sum(lens)), causal=causal, window=window)


@pytest.mark.parametrize("causal", [True, False])
def test_many_rows_that_see_nothing(dev, many_rows, causal):
    test_rows_that_see_nothing_are_zero(dev, causal)


def test_many_rows_scales_and_nan(dev, many_rows):
    test_scales_far_apart_and_peaked_scores(dev)
    test_nan_where_rows_do_not_look_stays_there(dev)
    test_nan_and_infinite_queries_and_scales(dev)


@pytest.mark.parametrize("rows,lens,window", [([5], [200], 0), ([150, 3], [200, 150], 40)])
def test_many_rows_a_scale_of_nan(dev, many_rows, rows, lens, window):
    test_a_scale_of_nan_reaches_only_rows_that_see_its_block(dev, rows, lens, window)


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("shape", ["rise", "fall", "spike", "late"])
def test_many_rows_scores_that_move_the_reference(dev, many_rows, page, rows, shape):
    test_scores_that_move_the_reference(dev, page, rows, shape)


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("rows,lens,heads,group,kw", [
    ([300, 257], [9001, 4200], 7, 1, {}),  # page numbers loaded more than once
    ([300], [9001], 14, 1, dict(causal=False, split_keys=False)),
    ([300, 1], [9001, 8000], 7, 1, dict(window=5000)),
    ([1100], [1100], 8, 1, {}),
])
def test_many_rows_long_key_ranges(dev, page, rows, lens, heads, group, kw):
    test_long_key_ranges_and_forms_in_between(dev, page, rows, lens, heads, group, kw)


def test_many_rows_bad_metadata(dev, many_rows):
    for rows in ([2, 3, 1], [150, 10, 20]):
        c = Case(dev, rows, [200, 190, 180], page=32, seed=41)
        clean, s = c.attend(), c.starts
        keep = c.plan.page_table[1, 2].clone()
        for bad in (-5, 10 ** 9):
            c.plan.page_table[1, 2] = bad
            got = c.attend()
            assert got[s[1]:s[2]].isnan().all()
            assert torch.equal(got[:s[1]], clean[:s[1]]) and torch.equal(got[s[2]:], clean[s[2]:])
        c.plan.page_table[1, 2] = keep
        for bad in (-1, 201, 2 ** 31 - 1):
            c.plan.kv_len[1] = bad
            got = c.attend()
            assert got[s[1]:s[2]].isnan().all()
            assert torch.equal(got[:s[1]], clean[:s[1]]) and torch.equal(got[s[2]:], clean[s[2]:])
        c.plan.kv_len[1] = 190
        assert torch.equal(c.attend(), clean)


@pytest.mark.parametrize("rows,lens", [([30], [700]), ([600], [900])])
def test_many_rows_out_may_be_q(dev, many_rows, rows, lens):
    from diffsynth_engine_amd import ops

    c = Case(dev, rows, lens, group=3, seed=rows[0])
    q = c.longer(c.q)
    assert ops.kv_attention(q, c.cache, c.plan, out=q) is q
    assert torch.equal(q[:c.total], c.attend()) and q[c.total:].isnan().all()
