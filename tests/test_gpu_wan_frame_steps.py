"""Wan frame by frame: the denoising steps of a run leave in the cache what its last step alone would have left, also in
the page that the run shares with finished frames.  Bits are compared: the kernels sum in a fixed order."""
import pytest
import torch

from oracle import wan as ow

pytestmark = pytest.mark.gpu


def _runner(dev, seed=1):
    from diffsynth_engine_amd.wan_dit import WanDiTRunner

    cfg = dict(ow.config_14b(), dim=512, ffn_dim=1024, num_heads=4, num_layers=2)
    return WanDiTRunner(ow.init_params(cfg, dtype=torch.bfloat16, seed=seed, bias_std=0.02), cfg, scaled=True, device=dev)


def _inputs(dev, frames, batch=1, seed=4):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, 16, frames, 12, 14, generator=g).bfloat16()  # 42 tokens a frame
    return x.to(dev), torch.randn(batch, 32, 4096, generator=g).bfloat16().to(dev), torch.full((batch,), 500.0).bfloat16().to(dev)


def _state(cache):
    return [t.view(torch.uint8).clone() for c in cache.layers for t in (c.k, c.v, c.k_scale, c.v_scale)]


@pytest.mark.parametrize("page,batch", [(64, 1), (16, 2)])
def test_the_steps_before_leave_nothing(dev, page, batch):
    R = _runner(dev)
    x, ctx, t = _inputs(dev, 4, batch)
    weights = [R.vec["blocks.%d.self_attn.norm_k.weight" % i] for i in range(2)]
    once, often = (R.frame_cache(4, 12, 14, batch=batch, page_size=page) for _ in range(2))
    for first, n in ((0, 2), (2, 1), (3, 1)):
        part = x[:, :, first:first + n].contiguous()
        for size in (1.0, 2.0 ** 14, 64.0):  # steps that are thrown away, their keys up to 2^14 times as large
            for w in weights:
                w.mul_(size)
            R(part.flip(3), ctx, t, cache=often, first_frame=first)
            for w in weights:
                w.div_(size)
        a = R(part, ctx, t, cache=once, first_frame=first)
        b = R(part, ctx, t, cache=often, first_frame=first)
        assert torch.equal(a, b), first
        # what a step writes beyond its own tokens is not read: compare what the cache holds
        tokens = (first + n) * 42
        for p, q in zip(once.layers, often.layers):
            for name in "kv":
                u, v = (getattr(c, name).view(torch.uint8).unflatten(0, (batch, -1)).transpose(2, 3).flatten(1, 2)[:, :tokens]
                        for c in (p, q))
                assert torch.equal(u, v), (first, name)
                u, v = (getattr(c, name + "_scale").view(torch.uint8).unflatten(0, (batch, -1))[:, :-(-tokens // page)]
                        for c in (p, q))
                assert torch.equal(u, v), (first, name)


def test_recorded_steps(dev):
    from diffsynth_engine_amd.graph import GraphedStep

    R = _runner(dev)
    x, ctx, t = _inputs(dev, 3)
    eager, replayed = (R.frame_cache(3, 12, 14) for _ in range(2))
    for c in (eager, replayed):
        R(x[:, :, :2].contiguous(), ctx, t, cache=c)
    part = x[:, :, 2:].contiguous()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(graph):
            replayed.step(2, 1)
    step = GraphedStep(R, x=part, context=ctx, timestep=t, cache=replayed, first_frame=2)
    for i in range(4):
        y = (part * (i + 1) * 0.5).contiguous()
        want = R(y, ctx, t, cache=eager, first_frame=2)
        torch.cuda.synchronize()
        assert torch.equal(step(x=y), want), i
        assert all(torch.equal(a, b) for a, b in zip(_state(eager), _state(replayed)))


def test_a_step_that_raises_leaves_no_frames_that_it_overwrote(dev, monkeypatch):
    R = _runner(dev)
    x, ctx, t = _inputs(dev, 3)
    cache, twin = (R.frame_cache(3, 12, 14) for _ in range(2))
    for c in (cache, twin):
        R(x, ctx, t, cache=c)
    block = R.block

    def stops(i, *args, **kw):
        if i == 1:
            raise KeyboardInterrupt
        return block(i, *args, **kw)

    part = x[:, :, 1:2].contiguous()
    monkeypatch.setattr(R, "block", stops)
    with pytest.raises(KeyboardInterrupt):
        R(part, ctx, t, cache=cache, first_frame=1)
    monkeypatch.undo()
    assert cache.frames == 1
    with pytest.raises(ValueError):  # frame 1 is not there any more
        R(x[:, :, 2:].contiguous(), ctx, t, cache=cache, first_frame=2)
    assert torch.equal(R(part, ctx, t, cache=cache, first_frame=1), R(part, ctx, t, cache=twin, first_frame=1))


def test_a_refused_call_leaves_the_run_in_progress_as_it_was(dev):
    R = _runner(dev)
    x, ctx, t = _inputs(dev, 3)
    once, often = (R.frame_cache(3, 12, 14) for _ in range(2))
    weights = [R.vec["blocks.%d.self_attn.norm_k.weight" % i] for i in range(2)]
    for c in (once, often):
        R(x[:, :, :1].contiguous(), ctx, t, cache=c)
        R(x[:, :, 1:2].contiguous(), ctx, t, cache=c, first_frame=1)
    part = x[:, :, 2:].contiguous()
    for w in weights:
        w.mul_(2.0 ** 14)
    R(part, ctx, t, cache=often, first_frame=2)  # a step that is thrown away
    for w in weights:
        w.div_(2.0 ** 14)
    state = _state(often)
    for bad in (dict(context=ctx[..., :100]), dict(x=part[:, :8])):  # a text width and a channel number that do not fit
        with pytest.raises(Exception):
            R(**{**dict(x=part, context=ctx, timestep=t, cache=often, first_frame=1), **bad})
    assert often.frames == 3 and all(torch.equal(a, b) for a, b in zip(state, _state(often)))
    assert torch.equal(R(part, ctx, t, cache=once, first_frame=2), R(part, ctx, t, cache=often, first_frame=2))
