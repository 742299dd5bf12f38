"""WanFrameCache's bookkeeping on host tensors: what a run's further steps find in the page that the run begins in."""
import pytest
import torch


def _cache(**kw):
    from diffsynth_engine_amd.wan_dit import WanFrameCache

    args = dict(layers=2, heads=3, frames=6, h=6, w=7, batch=2, page_size=64, device="cpu")
    args.update(kw)
    return WanFrameCache(**args)


def _write(cache, first, frames, value):
    """What a step leaves in the pages it appends to, whole blocks of one byte: new scales, kept codes rounded again."""
    for c in cache.layers:
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            t = t.view(torch.uint8).unflatten(0, (cache.batch, -1))
            t[:, first * 42 // 64:-(-(first + frames) * 42 // 64)] = value
    cache.frames = first + frames


def _state(cache):
    return [t.view(torch.uint8).clone() for c in cache.layers for t in (c.k, c.v, c.k_scale, c.v_scale)]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_further_step_begins_with_the_page_as_it_was_before_the_run():
    c = _cache()
    c.step(0, 2)
    _write(c, 0, 2, 11)          # 84 tokens: the second page is shared with the next run
    before = _state(c)
    c.step(2, 2)
    assert _same(_state(c), before)
    for value in (22, 33):       # steps of the run, each over a page as it was before the first
        _write(c, 2, 2, value)
        c.step(2, 2)
        for got, want in zip(_state(c), before):
            got, want = (t.unflatten(0, (2, -1)) for t in (got, want))
            assert torch.equal(got[:, :2], want[:, :2]) and (got[:, 2] == value).all()
    _write(c, 2, 2, 44)
    c.step(4, 1)
    _write(c, 4, 1, 55)
    c.step(2, 1)                 # back to an earlier run: its own copy
    for got, want in zip(_state(c), before):
        assert torch.equal(got.unflatten(0, (2, -1))[:, :2], want.unflatten(0, (2, -1))[:, :2])
    _write(c, 2, 2, 66)
    now = _state(c)
    c.step(4, 1)                 # the run behind it begins anew, over what is there now
    assert _same(_state(c), now)
    _write(c, 4, 1, 77)
    c.step(4, 1)
    for got, want in zip(_state(c), now):
        assert torch.equal(got.unflatten(0, (2, -1))[:, 2], want.unflatten(0, (2, -1))[:, 2])


def test_runs_that_begin_with_a_page_copy_nothing():
    c = _cache(h=8, w=8)
    c.step(0, 1)
    _write(c, 0, 1, 11)
    now = _state(c)
    c.step(1, 1)
    c.step(1, 1)
    assert _same(_state(c), now) and not c._before


def test_two_runs_in_one_page():
    c = _cache(h=2, w=5, batch=1)
    pages = lambda: _state(c)[0][0].flatten()[0].item()  # noqa: E731

    def write(first, value):
        for x in c.layers:
            x.k.view(torch.uint8)[0] = value
        c.frames = first + 1

    for first, value in ((0, 1), (1, 2), (2, 3)):
        c.step(first, 1)
        write(first, value)
    c.step(2, 1)
    assert pages() == 2
    write(2, 4)
    c.step(1, 1)
    assert pages() == 1


def test_layers_lie_apart_and_page_sizes_are_checked():
    c = _cache()
    for n, layer in enumerate(c.layers):
        assert layer.pages == 2 * 4 and layer.heads == 3 and layer.page_size == 64
        layer.k.view(torch.uint8).fill_(2 * n), layer.v.view(torch.uint8).fill_(2 * n + 1)
    assert all((c.layers[n].k.view(torch.uint8) == 2 * n).all() and (c.layers[n].v.view(torch.uint8) == 2 * n + 1).all()
               for n in range(2))
    with pytest.raises(ValueError):
        _cache(page_size=48)
