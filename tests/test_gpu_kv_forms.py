"""The paged cache's attention: limits of its number formats, and every form of its kernels on purpose.

A form is told from outside by the workspace that a call asks for: 520 bytes a row of a partial result, in 16- or 32-row
columns for the streaming form, 256 rows for the tile form, two for every compute unit where all tiles are shared evenly."""
import math

import pytest
import torch

from oracle import kv_cache as okv
from test_gpu_kv_cache import Case, ManyRows

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
