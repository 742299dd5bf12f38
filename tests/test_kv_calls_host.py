"""What ops.kv_append and ops.kv_attention refuse, and what they hand to the library, on the host: the device is replaced
by host tensors and the library by one that writes down its calls."""
import contextlib
import itertools
import random

import pytest
import torch

BF = torch.bfloat16


class Recorder:
    """Stands in for the library: every function notes the current device and returns 0."""

    def __init__(self):
        self.calls = []
        self.device = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, self.device))
            return 0
        return call


@pytest.fixture
def calls(monkeypatch):
    """ops with host tensors that pass for device 1's while device 0 is current."""
    from diffsynth_engine_amd import _lib, ops

    rec = Recorder()

    @contextlib.contextmanager
    def on(index):
        old, rec.device = rec.device, index
        yield
        rec.device = old

    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(ops, "_kv_device", lambda *a: 1)
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: rec.device, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    return rec


def _batch(heads=2, rows=6):
    from diffsynth_engine_amd.kv_cache import KVCache, KVPlan

    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return (KVCache.empty(4, heads, 16, "cpu"),
            KVPlan(torch.arange(4, dtype=torch.int32)[None], i32(0, rows), i32(40), max_rows=rows, max_kv_len=64))


def _elements(view):
    return set((view.data_ptr() // 2 + i * view.stride(0) + j * view.stride(1) + e)
               for i in range(view.shape[0]) for j in range(view.shape[1]) for e in range(128))


def test_views_meet_where_their_elements_do():
    from diffsynth_engine_amd.ops import _kv_meet

    r = random.Random(3)
    buf = torch.empty(60000, dtype=BF)
    seen = {True: 0, False: 0}
    for _ in range(400):
        views = []
        for _ in range(2):
            rows, heads = r.randrange(1, 6), r.randrange(1, 5)
            sh = r.choice((128, 128, 136, 256, 384, 1280))
            sr = r.choice((128 * heads, 1280, 1280, 640, 128, 2560, 1288))
            at = 8 * r.randrange(0, 700)
            views.append(buf.as_strided((rows, heads, 128), (sr, sh, 1), at))
        for a, b in (views, views[::-1]):
            got = _kv_meet(*((t.data_ptr(), t.stride(0), t.stride(1), *t.shape[:2]) for t in (a, b)))
            assert got == bool(_elements(a) & _elements(b)), (a.shape, a.stride(), b.shape, b.stride())
            seen[got] += 1
    assert min(seen.values()) > 100
    for shape in ((0, 3, 128), (3, 0, 128)):
        t = buf.as_strided(shape, (384, 128, 1))
        assert not _kv_meet(*((t.data_ptr(), 384, 128, *shape[:2]) for _ in range(2)))


def test_outputs_over_inputs_are_refused(calls):
    from diffsynth_engine_amd import ops

    cache, plan = _batch()
    packed = torch.zeros(8, 8, 128, dtype=BF)
    q, k, v = packed[:6, :4], packed[:6, 4:6], packed[:6, 6:]
    row_on, head_on = packed[1:7, :4], packed[:6, 1:5]
    far = torch.empty_like(packed)
    for bad in (row_on, head_on):
        with pytest.raises(ValueError, match="overlaps"):
            ops.kv_attention(q, cache, plan, out=bad)
    for bad in (row_on, head_on, packed[:6, 2:6], packed[:6, 4:], packed[2:, 3:7]):
        with pytest.raises(ValueError, match="overlaps"):
            ops.kv_append(k, v, cache, plan, q=q, q_out=bad)
    with pytest.raises(ValueError, match="overlaps"):  # q itself, but k is a part of it
        ops.kv_append(q[:, 1:3], v, cache, plan, q=q, q_out=q)
    assert not calls.calls
    for good in (q, far[:6, :4], far[2:, 1:5], far[:6, ::2]):
        assert ops.kv_attention(q, cache, plan, out=good) is good
        assert ops.kv_append(k, v, cache, plan, q=q, q_out=good) is good
    assert ops.kv_attention(q, cache, plan, out=packed[:6, 4:]) is not None  # what is not read here may be written
    wide = torch.zeros(6, 8, 128, dtype=BF)
    for a, b in itertools.permutations((wide[:, ::2], wide[:, 1::2])):  # every other head of one buffer
        assert ops.kv_attention(a, cache, plan, out=b) is b
    one = wide[:1, :1]
    assert ops.kv_attention(one, _batch(1, 1)[0], plan, out=one.as_strided((1, 1, 128), (8, 8, 1))) is not None


def test_a_scale_whose_base_2_form_is_infinite_is_refused(calls):
    # fp32's largest number over log2(e) is 2.36e38: beyond it 0 * infinity made NaN of a score of zero
    from diffsynth_engine_amd import ops

    cache, plan = _batch()
    q = torch.zeros(6, 2, 128, dtype=BF)
    for bad in (2.3e38, 2.9e38):
        with pytest.raises(ValueError, match="scale"):
            ops.kv_attention(q, cache, plan, scale=bad)
    assert not calls.calls
    ops.kv_attention(q, cache, plan, scale=2.2e38)


def test_the_library_refuses_it_too():
    import ctypes

    from diffsynth_engine_amd import _lib

    cache, plan = _batch()
    for scale, need in ((2.3e38, True), (2.4e38, False), (3.4e38, False)):
        P = _lib.KVAttnParams(total_rows=6, softmax_scale=scale, heads_q=2)
        long = type(plan._c).from_buffer_copy(plan._c)
        long.max_kv_len, long.table_pages, long.table_sb = 1 << 20, 1 << 16, 1 << 16
        got = _lib.load().dsx_kv_attn_workspace_bytes(ctypes.byref(cache._c), ctypes.byref(long), ctypes.byref(P))
        assert (got > 0) == need  # (0 for a call that would be refused)


def test_the_workspace_is_sized_by_the_tensors_device(calls):
    # how a call is split depends on the compute units of the device that it runs on
    from diffsynth_engine_amd import ops

    cache, plan = _batch()
    ops.kv_attention(torch.zeros(6, 2, 128, dtype=BF), cache, plan)
    assert calls.calls == [("dsx_kv_attn_workspace_bytes", 1), ("dsx_kv_attn", 1)] and calls.device == 0
    calls.calls.clear()
    ops.kv_attention(torch.zeros(6, 2, 128, dtype=BF), cache, plan, split_keys=False)
    assert calls.calls == [("dsx_kv_attn", 1)]


@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
def test_plan_check_looks_at_the_scales_of_pages_that_hold_tokens(name):
    from diffsynth_engine_amd.kv_cache import KVCache, KVPlan

    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    cache = KVCache.empty(6, 3, 16, "cpu")
    # sequence 0: 20 tokens, 3 of them rows, on pages 4 and 1; sequence 1: 17 tokens, all rows, on 2 and 0
    plan = KVPlan(i32([[4, 1, -7], [2, 0, 99]]), i32([0, 3, 20]), i32([20, 17]), max_rows=17, max_kv_len=48)
    raw = getattr(cache, name).view(torch.uint8)
    for page, append, attend in ((4, 0, 0), (1, 0, 0), (2, None, 1), (0, None, 1), (3, None, None), (5, None, None)):
        for value, fits in ((78, False), (79, True), (175, True), (176, False), (254, False), (0, False), (255, True)):
            raw[page, 2] = value
            for for_append, bad in ((True, append), (False, attend)):
                if fits or bad is None:
                    plan.check(cache, 20, for_append=for_append)
                else:
                    with pytest.raises(ValueError, match=r"sequence %d \(page %d\)" % (bad, page)):
                        plan.check(cache, 20, for_append=for_append)
        raw[page, 2] = 127
    plan.kv_len.copy_(i32([3, 17]))  # no tokens before the rows: nothing to look at
    raw.fill_(0)
    plan.check(cache, 20)
    # strided scales
    wide = torch.full((6, 2, 3), 127, dtype=torch.uint8)
    wide[:, 1] = 0
    args = dict(k_scale=cache.k_scale, v_scale=cache.v_scale)
    for t in args.values():
        t.view(torch.uint8).fill_(127)
    args[name] = wide[:, 0].view(torch.float8_e8m0fnu)
    plan.check(KVCache(cache.k, cache.v, **args), 20, for_append=False)


@pytest.mark.parametrize("seqs,rows,heads,group,tokens,window,form", [
    (1, 1, 12, 1, 1561, 0, (1, 12 * 6)),            # few units: equal pieces, as many as there are compute units and tiles
    (32, 1, 8, 4, 4097, 0, None),                   # a unit for every compute unit: uncut
    (64, 1, 8, 4, 16384, 0, (1, 512)),              # long: two partial results for every compute unit
    (64, 1, 8, 4, 4064, 0, None), (64, 1, 8, 4, 8160, 0, (1, 512)),
    (64, 5, 8, 4, 16384, 0, (2, 512)), (64, 5, 8, 4, 16384, 4000, None), (64, 5, 8, 4, 16384, 12000, (2, 512)),
    (1, 1, 40, 1, 131071, 0, (1, 512)), (1, 4, 40, 7, 131072, 0, (2, 512)), (40, 32, 8, 1, 16384, 0, (2, 512)),
    (700, 1, 8, 17, 1024, 0, (2, 512)),
    (8, 5, 4, 7, 20000, 4096, (2, 64 * 4)),         # two blocks of two columns
    (1, 600, 12, 1, 2048, 0, None),                 # many blocks, a short cache
    (2, 300, 1, 1, 9001, 0, (2, 20 * 12)), (1, 300, 1, 1, 9001, 0, (2, 10 * 25)),  # many rows and still the streaming form
    (2, 300, 7, 1, 9001, 0, (16, 28 * 9)),          # the tile form, all of its units cut
    (1, 1560, 40, 1, 10920, 0, (16, 24 * 10)),      # and those behind a whole round
    (1, 4680, 40, 1, 32760, 0, None),               # 760 units on 256: 248 behind two rounds, too many to cut
    (3, 4096, 8, 4, 5001, 0, None),
])
def test_which_form_a_call_takes(seqs, rows, heads, group, tokens, window, form):
    """(16-row columns of a partial result, their number) by the workspace that the call asks for; None: nothing is cut.  The
    host's answer where no device can be asked is that of 256 compute units."""
    import ctypes

    from diffsynth_engine_amd import _lib

    if torch.cuda.is_available() and torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("another number of compute units")
    at = 1 << 20  # nothing is launched, and no pointer followed
    C = _lib.KVCacheParams(k=at, v=at, k_scale=at, v_scale=at, k_sp=heads * 8192, k_sh=8192, v_sp=heads * 8192, v_sh=8192,
                           ks_sp=heads, vs_sp=heads, pages=100, heads=heads, page_size=64)
    N = _lib.KVBatchParams(page_table=at, table_sb=4096, row_start=at, kv_len=at, batch=seqs, table_pages=4096,
                           max_rows=rows, max_kv_len=tokens)
    P = _lib.KVAttnParams(total_rows=seqs * rows, softmax_scale=0.1, heads_q=heads * group, window=window)
    got = _lib.load().dsx_kv_attn_workspace_bytes(ctypes.byref(C), ctypes.byref(N), ctypes.byref(P))
    assert got == (0 if form is None else form[0] * 16 * form[1] * 520)
