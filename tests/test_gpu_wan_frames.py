"""Wan frame by frame: runs of frames over an 8-bit cache of the frames in front of them, against the oracle's block with
a mask over the whole sequence and keys and values rounded as the cache rounds them (the same criterion as the block and
step tests without a cache)."""
import pytest
import torch

from oracle import kv_cache as okv
from oracle import wan as ow

pytestmark = pytest.mark.gpu


def _cos(a, b):
    return torch.nn.functional.cosine_similarity(a.float().flatten().cpu(), b.float().flatten().cpu(), dim=0).item()


def _rounded(x, page, bounds):
    """(S, H, 128) as the cache holds it after appends that end at `bounds`."""
    S, H, _ = x.shape
    pages = -(-S // page)
    cache = {n: torch.zeros(pages, H, page, 128).to(torch.float8_e4m3fn) for n in "kv"}
    cache.update({n + "_scale": torch.zeros(pages, H, dtype=torch.int32) for n in "kv"})
    at = 0
    for end in bounds:
        new = okv.append(cache, [list(range(pages))], [0, end - at], [end], x[at:end], x[at:end])
        for n in "kv":
            cache[n], cache[n + "_scale"] = okv.e4m3_nearest(new[n][0]).float().to(torch.float8_e4m3fn), new[n][1]
        at = end
    return okv.values(cache["v"], cache["v_scale"]).transpose(1, 2).flatten(0, 1)[:S].to(x.dtype)


def _masked_attention(tokens, runs, page):
    """The oracle's attention callable: self-attention calls (as many keys as queries) see whole runs up to their own,
    over rounded keys and values; others are left alone."""
    bounds = [sum(runs[:i + 1]) * tokens for i in range(len(runs))]
    run_of = torch.repeat_interleave(torch.arange(len(runs)), torch.tensor(runs) * tokens)

    def attn(q, k, v):
        if k.shape[2] != q.shape[2]:
            return ow.O.sdpa(q, k, v)
        out = []
        for b in range(q.shape[0]):
            kk, vv = (_rounded(t[b].transpose(0, 1), page, bounds).transpose(0, 1) for t in (k, v))
            s = q[b].float() @ kk.float().transpose(1, 2) / 128 ** 0.5
            s = s.masked_fill(run_of[None, :, None] < run_of[None, None, :], float("-inf"))
            out.append((torch.softmax(s, -1) @ vv.float()).to(q.dtype))
        return torch.stack(out)

    return attn


def _small(seed=1):
    cfg = dict(ow.config_14b(), dim=512, ffn_dim=1024, num_heads=4, num_layers=2)
    return cfg, ow.init_params(cfg, dtype=torch.bfloat16, seed=seed, bias_std=0.02)


@pytest.mark.parametrize("runs,page,batch", [((2, 1, 2), 64, 1), ((1, 1, 1, 1), 16, 2), ((5,), 32, 1)])
def test_block_in_runs_of_frames(dev, runs, page, batch):
    from diffsynth_engine_amd.wan_dit import WanDiTRunner

    cfg, sd = _small()
    g = torch.Generator().manual_seed(2)
    f, h, w = sum(runs), 6, 7
    x = torch.randn(batch, f * h * w, 512, generator=g).bfloat16()
    ctx = torch.randn(batch, 40, 512, generator=g).bfloat16()
    t_mod = (torch.randn(1, 6, 512, generator=g) * 0.3).bfloat16()
    want = ow.dit_block(ow.Params(sd, "fp8_scaled"), 0, x, ctx, t_mod, ow.freqs_cis_3d(128, f, h, w), cfg,
                        attn=_masked_attention(h * w, runs, page))
    R = WanDiTRunner(sd, cfg, scaled=True, device=dev)
    cache = R.frame_cache(f, 2 * h, 2 * w, batch=batch, page_size=page)
    got, first = [], 0
    for n in runs:
        part = slice(first * h * w, (first + n) * h * w)
        plan = cache.plan(first, n)
        for _ in range(2):  # a second step over the same frames: the block's keys and values are written again
            y = R.block(0, x[:, part].to(dev), ctx.to(dev), t_mod.expand(batch, -1, -1).to(dev).contiguous(),
                        R.rope_table(n, h, w, first=first), kv=(cache.layers[0], plan))
        got.append(y.cpu())
        first += n
        cache.frames = first
    assert _cos(torch.cat(got, 1), want) >= 0.9995


def test_model_in_runs_of_frames(dev):
    from diffsynth_engine_amd.wan_dit import WanDiTRunner

    cfg, sd = _small(seed=3)
    g = torch.Generator().manual_seed(4)
    runs, page = (2, 1), 64
    x = torch.randn(1, 16, 3, 12, 16, generator=g).bfloat16()
    ctx = torch.randn(1, 32, 4096, generator=g).bfloat16()
    t = torch.tensor([500.0]).bfloat16()
    P = ow.Params(sd, "fp8_scaled")
    want = ow.wan_dit_forward(P, x, ctx, t, cfg, attn=_masked_attention(48, runs, page))
    nudged = x.clone()
    nudged.view(torch.int16).flatten()[::64] ^= 1
    floor = _cos(want, ow.wan_dit_forward(P, nudged, ctx, t, cfg, attn=_masked_attention(48, runs, page)))
    R = WanDiTRunner(sd, cfg, scaled=True, device=dev)
    cache = R.frame_cache(3, 12, 16, page_size=page)
    got, first = [], 0
    for n in runs:
        for _ in range(2):
            y = R(x[:, :, first:first + n].to(dev), ctx.to(dev), t.to(dev), cache=cache, first_frame=first)
        got.append(y.cpu())
        first += n
    assert cache.frames == 3 and cache.bytes() == 2 * 2 * (3 * 64 * 4 * 128 + 3 * 4)
    c = _cos(torch.cat(got, 2), want)
    assert c >= 0.99 and c >= min(0.999, floor - 2e-3), (c, floor)


def test_frames_refuse_what_does_not_fit(dev):
    from diffsynth_engine_amd.wan_dit import WanDiTRunner

    cfg, sd = _small()
    R = WanDiTRunner(sd, cfg, scaled=True, device=dev)
    cache = R.frame_cache(3, 12, 16)
    x = torch.randn(1, 16, 2, 12, 16, device=dev).bfloat16()
    ctx, t = torch.randn(1, 8, 4096, device=dev).bfloat16(), torch.tensor([500.0], device=dev).bfloat16()
    for bad in (dict(first_frame=1), dict(cache=cache, first_frame=1), dict(cache=cache, first_frame=-1),
                dict(cache=R.frame_cache(1, 12, 16)), dict(cache=R.frame_cache(3, 12, 14)),
                dict(cache=R.frame_cache(3, 12, 16, batch=2))):
        with pytest.raises(ValueError):
            R(x, ctx, t, **bad)
    R(x, ctx, t, cache=cache)
    with pytest.raises(ValueError):
        R(x, ctx, t, cache=cache, first_frame=2)  # frames 2 and 3 of three
    with pytest.raises(ValueError):
        R.frame_cache(0, 12, 16)
