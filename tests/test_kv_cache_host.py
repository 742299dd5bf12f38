"""The paged key/value cache on the host: struct layouts, argument checks that need no GPU, the bounds of a plan, and
the oracle against known answers."""
import ctypes
import math
import os
import re

import pytest
import torch

from oracle import kv_cache as okv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, F8, E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _cache(pages=4, heads=2, page=16):
    from diffsynth_engine_amd.kv_cache import KVCache

    return KVCache.empty(pages, heads, page, device="cpu")


def _plan(table=((0, 1), (2, -1)), starts=(0, 3, 4), lens=(20, 7), max_rows=4, max_kv_len=32):
    from diffsynth_engine_amd.kv_cache import KVPlan

    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return KVPlan(i32(table), i32(starts), i32(lens), max_rows=max_rows, max_kv_len=max_kv_len)


@pytest.mark.parametrize("struct,name", [("dsx_kv_cache", "KVCacheParams"), ("dsx_kv_batch", "KVBatchParams"),
                                         ("dsx_kv_append_params", "KVAppendParams"),
                                         ("dsx_kv_attn_params", "KVAttnParams")])
def test_struct_layouts_match_the_header(struct, name):
    from diffsynth_engine_amd import _lib

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "dsx.h")).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
    want = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        first, *more = [x.strip() for x in decl.split(",")]
        ctype, _, field = first.rpartition(" ")
        kind = ctypes.c_void_p if "*" in decl else {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32,
                                                    "float": ctypes.c_float}[ctype.replace("const", "").strip()]
        want += [(f.strip("* "), kind) for f in [field] + more]
    assert list(getattr(_lib, name)._fields_) == want


def test_cache_refuses_what_does_not_fit():
    from diffsynth_engine_amd.kv_cache import KVCache

    c = _cache()
    good = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale)
    KVCache(**good)
    wide = torch.zeros(4, 2, 16, 256, dtype=torch.uint8).view(F8)
    for bad in (dict(v=c.v[:2]), dict(k=c.k.view(torch.uint8)), dict(k=c.k.float()), dict(k=wide[..., :128]),
                dict(k=c.k[:, :, :8], v=c.v[:, :, :8]), dict(k=c.k[..., :64], v=c.v[..., :64]),
                dict(k=c.k[:0], v=c.v[:0], k_scale=c.k_scale[:0], v_scale=c.v_scale[:0]),
                dict(k_scale=c.k_scale[:, :1]), dict(v_scale=torch.ones(4, 2)),
                dict(k_scale=c.k_scale.view(torch.uint8).t().contiguous().t().view(E8)),
                dict(k=c.k.view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(F8))):
        with pytest.raises(ValueError):
            KVCache(**{**good, **bad})
    for page in (0, 8, 48, 256):
        with pytest.raises(ValueError):
            KVCache.empty(2, 1, page, device="cpu")
    # k and v as two slices of one buffer: page strides of their own
    both = torch.zeros(4, 2, 2, 16, 128, dtype=torch.uint8).view(F8)
    assert KVCache(both[:, 0], both[:, 1], c.k_scale, c.v_scale)._c.k_sp == 2 * 2 * 16 * 128


def test_cache_and_plan_are_fixed_and_blocks_lie_apart():
    from diffsynth_engine_amd.kv_cache import KVCache

    c, plan = _cache(), _plan()
    for thing, name in ((c, "k"), (c, "v_scale"), (c, "page_size"), (plan, "kv_len"), (plan, "max_kv_len")):
        with pytest.raises(AttributeError):
            setattr(thing, name, getattr(thing, name))
    k, s = c.k.view(torch.uint8), c.k_scale.view(torch.uint8)
    for codes, scales in ((k[:1].expand(4, -1, -1, -1), s), (k[:, :1].expand(-1, 2, -1, -1), s), (k, s[:1].expand(4, -1)),
                          (k.as_strided((4, 2, 16, 128), (2048, 2048, 128, 1)), s), (k, s.as_strided((4, 2), (1, 1)))):
        with pytest.raises(ValueError):
            KVCache(codes.view(F8), c.v, scales.view(E8), c.v_scale)
    heads_outside = k.transpose(0, 1).contiguous().transpose(0, 1).view(F8)  # (pages, heads) stored the other way round
    assert KVCache(heads_outside, c.v, c.k_scale, c.v_scale)._c.k_sp == 2048
    every_other = torch.zeros(4, 3, 16, 128, dtype=torch.uint8)[:, ::2].view(F8)
    assert KVCache(every_other, c.v, c.k_scale, c.v_scale)._c.k_sh == 4096


def test_plan_refuses_what_does_not_fit():
    from diffsynth_engine_amd.kv_cache import KVPlan

    _plan()
    for bad in (dict(starts=(0, 3)), dict(lens=(20,)), dict(table=(0, 1)), dict(max_rows=-1), dict(max_kv_len=-1),
                dict(max_rows=2 ** 31), dict(max_kv_len=2 ** 31)):
        with pytest.raises(ValueError):
            _plan(**bad)
    t, s, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in ((t.long(), s, n), (t, s.long(), n), (t, s, n.float()), (t.t().contiguous().t(), s, n),
                (t, torch.zeros(6, dtype=torch.int32)[::2], n), (t[:1].expand(2, 2), s, n), (t[:, :0], s, n)):
        with pytest.raises(ValueError):
            KVPlan(*bad, max_rows=1, max_kv_len=1)
    with pytest.raises(ValueError):
        _plan(max_kv_len=33)._fits(_cache())  # two pages of 16


def test_host_tensors_are_refused_not_computed():
    from diffsynth_engine_amd import ops

    x = torch.zeros(4, 2, 128, dtype=BF)
    with pytest.raises(RuntimeError):
        ops.kv_append(x, x, _cache(), _plan())
    with pytest.raises(RuntimeError):
        ops.kv_attention(x, _cache(), _plan())


@pytest.mark.parametrize("append,kw,bad", [
    (True, dict(), None),
    (True, dict(lens=(2, 7)), 0),                               # three rows, two tokens
    (False, dict(lens=(2, 7)), None),                           # ... which attention takes
    (False, dict(lens=(20, -1)), 1), (False, dict(lens=(33, 7)), 0),
    (False, dict(starts=(0, 3, 2)), 1), (False, dict(starts=(-1, 3, 4)), 0), (False, dict(starts=(0, 3, 5)), 1),
    (False, dict(starts=(0, 0, 4), max_rows=3), 1),
    (False, dict(table=((0, 4), (2, 0))), 0), (False, dict(table=((0, 1), (-1, 0))), 1),
    (False, dict(table=((0, 1), (2, 99))), None),               # an entry that no token needs
    (False, dict(table=((0, 1), (1, -1))), None),               # a shared page is fine to read,
    (True, dict(table=((0, 1), (1, -1))), 0),                   # ... not to write
    (True, dict(table=((0, 1), (0, -1))), 1),                   # sequence 0 writes page 1 only, sequence 1 page 0
    (True, dict(table=((1, 1), (2, -1))), 0),
    (True, dict(starts=(0, 0, 4), table=((0, 1), (2, -1))), None),
])
def test_plan_check(append, kw, bad):
    plan = _plan(**kw)
    if bad is None:
        plan.check(_cache(), 4, for_append=append)
    else:
        with pytest.raises(ValueError, match="sequence %d " % bad):
            plan.check(_cache(), 4, for_append=append)


def test_c_entries_refuse_bad_calls_before_any_launch():
    from diffsynth_engine_amd import _lib

    lib = _lib.load()
    buf = ctypes.create_string_buffer(8192)
    at = (ctypes.addressof(buf) + 255) & ~255
    cache, plan = _cache(), _plan()

    def attn(c=None, n=None, **kw):
        P = _lib.KVAttnParams(q=at, q_sr=256, q_sh=128, out=at, o_sr=256, o_sh=128, total_rows=4, softmax_scale=0.1,
                              heads_q=2)
        for key, val in kw.items():
            setattr(P, key, val)
        return lib.dsx_kv_attn(ctypes.byref(c or cache._c), ctypes.byref(n or plan._c), ctypes.byref(P), None)

    def append(c=None, n=None, **kw):
        P = _lib.KVAppendParams(k=at, k_sr=256, k_sh=128, v=at, v_sr=256, v_sh=128, total_rows=4, norm_eps=1e-6)
        for key, val in kw.items():
            setattr(P, key, val)
        return lib.dsx_kv_append(ctypes.byref(c or cache._c), ctypes.byref(n or plan._c), ctypes.byref(P), None)

    def changed(s, **kw):
        t = type(s).from_buffer_copy(s)
        for key, val in kw.items():
            setattr(t, key, val)
        return t

    for call in (attn, append):
        for kw in (dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None)):
            assert call(c=changed(cache._c, **kw)) == _lib.DSX_ENULL
        for kw in (dict(page_table=None), dict(row_start=None), dict(kv_len=None)):
            assert call(n=changed(plan._c, **kw)) == _lib.DSX_ENULL
        for kw in (dict(page_size=24), dict(pages=0), dict(heads=0)):
            assert call(c=changed(cache._c, **kw)) == _lib.DSX_EBADSHAPE
        for kw in (dict(k_sp=2 ** 31), dict(v_sp=-2048), dict(ks_sp=2 ** 31), dict(vs_sp=-2)):
            assert call(c=changed(cache._c, **kw)) == _lib.DSX_EBADSHAPE
        assert call(n=changed(plan._c, table_sb=2 ** 31)) == _lib.DSX_EBADSHAPE
        for kw in (dict(k_sp=2056), dict(v_sh=8), dict(k=at + 8)):
            assert call(c=changed(cache._c, **kw)) == _lib.DSX_EALIGN
        for kw in (dict(batch=0), dict(table_pages=0), dict(table_sb=1), dict(max_rows=-1), dict(max_kv_len=33),
                   dict(max_kv_len=-1)):
            assert call(n=changed(plan._c, **kw)) == _lib.DSX_EBADSHAPE
        assert call(total_rows=-1) == _lib.DSX_EBADSHAPE
        assert call(total_rows=2 ** 31) == _lib.DSX_EBADSHAPE
        assert call(total_rows=0) == _lib.DSX_OK  # nothing to do, nothing launched
    for kw, rc in ((dict(q=None), _lib.DSX_ENULL), (dict(out=None), _lib.DSX_ENULL), (dict(q=at + 2), _lib.DSX_EALIGN),
                   (dict(o_sr=252), _lib.DSX_EALIGN), (dict(q_sr=2 ** 31), _lib.DSX_EALIGN), (dict(o_sh=-128), _lib.DSX_EALIGN), (dict(heads_q=3), _lib.DSX_EBADSHAPE),
                   (dict(heads_q=0), _lib.DSX_EBADSHAPE), (dict(window=-1), _lib.DSX_EBADSHAPE),
                   (dict(softmax_scale=0.0), _lib.DSX_EBADSHAPE), (dict(softmax_scale=math.nan), _lib.DSX_EBADSHAPE),
                   (dict(softmax_scale=math.inf), _lib.DSX_EBADSHAPE), (dict(softmax_scale=-1.0), _lib.DSX_EBADSHAPE),
                   (dict(workspace=at + 4), _lib.DSX_EALIGN)):
        assert attn(**kw) == rc, kw
    long = changed(plan._c, max_kv_len=1 << 20, table_pages=1 << 16, table_sb=1 << 16)
    P = _lib.KVAttnParams(total_rows=4, softmax_scale=0.1, heads_q=2)
    need = lib.dsx_kv_attn_workspace_bytes(ctypes.byref(cache._c), ctypes.byref(long), ctypes.byref(P))
    assert need > 0
    assert attn(n=long, workspace=at, workspace_bytes=need - 1) == _lib.DSX_EWORKSPACE
    for kw, rc in ((dict(k=None), _lib.DSX_ENULL), (dict(v=None), _lib.DSX_ENULL), (dict(q=at), _lib.DSX_ENULL),
                   (dict(q=at, q_out=at), _lib.DSX_EBADSHAPE), (dict(k=at + 2), _lib.DSX_EALIGN),
                   (dict(v_sr=100), _lib.DSX_EALIGN), (dict(k_sh=-128), _lib.DSX_EALIGN), (dict(q=at, q_out=at + 2, heads_q=1), _lib.DSX_EALIGN),
                   (dict(k_norm_w=at + 2), _lib.DSX_EALIGN), (dict(norm_eps=-1.0), _lib.DSX_EBADSHAPE),
                   (dict(norm_eps=math.nan), _lib.DSX_EBADSHAPE), (dict(rope=at, rope_rows=31), _lib.DSX_EBADSHAPE),
                   (dict(rope=at, rope_rows=32, rope_sb=128), _lib.DSX_EBADSHAPE)):
        assert append(**kw) == rc, kw
    # bounds that no launch could cover
    large = changed(plan._c, batch=1 << 23, max_rows=4)
    assert attn(n=large) == _lib.DSX_EBADSHAPE and append(n=large) == _lib.DSX_EBADSHAPE
    rows = changed(plan._c, batch=1 << 12, max_rows=1 << 20, max_kv_len=1 << 20, table_pages=1 << 16, table_sb=1 << 16)
    assert append(n=rows, total_rows=1 << 20) == _lib.DSX_EBADSHAPE
    assert attn(n=rows, total_rows=1 << 20) == _lib.DSX_EBADSHAPE


def test_oracle_rounding_against_torch_and_known_answers():
    bits = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(BF)
    x = bits[torch.isfinite(bits) & (bits.abs() <= 448)]
    assert torch.equal(okv.e4m3_nearest(x.double()).float(), x.to(F8).float())
    assert okv.e4m3_nearest(torch.tensor([1e9, -math.inf, 464.0], dtype=torch.float64)).tolist() == [448, -448, 448]
    assert [okv.block_exponent(a) for a in (0.0, 448.0, 448.0001, 224.0, 1.75, 1.76, 1e30, 1e-30)] == \
        [-48, 0, 1, -1, -8, -7, 48, -48]


def test_oracle_attention_against_sdpa():
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(23, 2, 128, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(5, 4, 128, generator=g).bfloat16()
    cache = {n: torch.zeros(2, 2, 16, 128).to(F8) for n in "kv"}
    cache.update({n + "_scale": torch.zeros(2, 2, dtype=torch.int32) for n in "kv"})
    new = okv.append(cache, [[1, 0]], [0, 23], [23], k, v)
    for n in "kv":
        cache[n], cache[n + "_scale"] = okv.e4m3_nearest(new[n][0]).float().to(F8), new[n][1]
    kk, vv = (okv.values(cache[n], cache[n + "_scale"])[[1, 0]].transpose(0, 1).flatten(1, 2)[:, :23] for n in "kv")
    assert ((kk.transpose(0, 1) - k.double()).abs() <= 2.0 ** -4 * k.double().abs() + 2.0 ** -16).all()
    mask = torch.arange(23)[None] <= torch.arange(5)[:, None] + 18
    want = torch.nn.functional.scaled_dot_product_attention(
        q.double().transpose(0, 1), kk.repeat_interleave(2, 0), vv.repeat_interleave(2, 0), attn_mask=mask)
    got, _ = okv.attention(q, cache, [[1, 0]], [0, 5], [23])
    assert torch.allclose(got.transpose(0, 1), want, atol=1e-12)
