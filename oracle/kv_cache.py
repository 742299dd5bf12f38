"""The paged 8-bit key/value cache in 64 bits, one sequence and head at a time — oracle (test infrastructure, see
oracle/__init__.py).  Nothing in the reference corresponds to it; the definitions are those of ``include/dsx.h``.

A cache here is a dict of CPU tensors: k, v (pages, heads, page, 128) e4m3; k_scale, v_scale (pages, heads) int exponents.
A batch is three lists: table (pages of every sequence), row_start, kv_len."""
import math

import torch

from .fp8 import e4m3_to_f32

D = 128


def e4m3_nearest(x: torch.Tensor) -> torch.Tensor:
    """float64 values -> the nearest e4m3 value (ties to the even code), saturating at +-448; NaN stays NaN."""
    a = x.abs().clamp(max=448.0)
    _, ex = torch.frexp(torch.where(a > 0, a, torch.ones_like(a)))
    step = torch.ldexp(torch.ones_like(a), (ex - 4).clamp(min=-9))  # 2^-9 below 2^-6: the subnormals
    # torch.round ties to even, as the mantissa does
    return torch.where(x.isnan(), x, torch.copysign(torch.round(a / step) * step, x))


def values(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """float64 values of (.., page, 128) codes with their block exponents."""
    f = torch.from_numpy(e4m3_to_f32(codes.contiguous().view(torch.uint8).numpy())).double()
    return f * torch.ldexp(torch.ones_like(exps, dtype=torch.float64), exps)[..., None, None]


def block_exponent(amax: float) -> int:
    """Smallest e in [-48, 48] with amax <= 448 * 2^e."""
    e = -48
    while e < 48 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def norm_rope(x: torch.Tensor, weight, rope, pos, eps=1e-6) -> torch.Tensor:
    """x (rows, heads, 128) -> float64; rope (positions, 64, 2)."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    if rope is not None:
        c, s = rope[pos].double().unbind(-1)
        a, b = x[..., 0::2], x[..., 1::2]
        x = torch.stack((a * c[:, None] - b * s[:, None], a * s[:, None] + b * c[:, None]), -1).flatten(-2)
    return x


def append(cache, table, row_start, kv_len, k, v, k_norm_w=None, rope=None, eps=1e-6):
    """Returns {name: (exact float64 values scaled to their block, exponents)} for k and v after the append: block
    (page, head) of the first holds value / 2^exponent before its rounding to e4m3."""
    page = cache["k"].shape[2]
    out = {}
    for name, x in (("k", k), ("v", v)):
        exps = cache[name + "_scale"].clone()
        scaled = values(cache[name], torch.zeros_like(exps))
        for b in range(len(kv_len)):
            r0, r1, n = row_start[b], row_start[b + 1], kv_len[b]
            first = n - (r1 - r0)
            part = x[r0:r1].double()
            if name == "k":
                part = norm_rope(part, k_norm_w, None if rope is None else rope[b if rope.shape[0] > 1 else 0],
                                 torch.arange(first, n), eps)
            for t0 in range(first // page * page, n, page) if r1 > r0 else ():
                lo, hi = max(first, t0), min(n, t0 + page)
                at = table[b][t0 // page]
                new = part[lo - first:hi - first]
                for h in range(x.shape[1]):
                    y = new[:, h]
                    fine = y[torch.isfinite(y)]
                    e = block_exponent(fine.abs().max().item() if fine.numel() else 0.0)
                    old = int(exps[at, h])
                    if lo > t0 and old > e:
                        e = old
                    if lo > t0 and e > old:
                        scaled[at, h, :lo - t0] *= 2.0 ** (old - e)
                    scaled[at, h, lo - t0:hi - t0] = (y * 2.0 ** -e).clamp(-448, 448)
                    exps[at, h] = e
        out[name] = (scaled, exps)
    return out


def attention(q, cache, table, row_start, kv_len, *, causal=True, window=0, scale=None):
    """(output, sum_j p_j |v_j|) in float64 for every packed row that belongs to a sequence; NaN rows elsewhere."""
    scale = 1 / math.sqrt(D) if scale is None else scale
    heads, page = cache["k"].shape[1:3]
    g = q.shape[1] // heads
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    size = out.clone()
    kk, vv = values(cache["k"], cache["k_scale"]), values(cache["v"], cache["v_scale"])
    for b in range(len(kv_len)):
        r0, r1, n = row_start[b], row_start[b + 1], kv_len[b]
        for i in range(r1 - r0):
            end = max(n - (r1 - r0) + i + 1, 0) if causal else n
            begin = max(end - window, 0) if window else 0
            if end <= begin:
                out[r0 + i] = size[r0 + i] = 0
                continue
            tok = torch.arange(begin, end)
            at = torch.tensor(table[b])[tok // page]
            for h in range(heads):
                ks, vs = kk[at, h, tok % page], vv[at, h, tok % page]
                p = torch.softmax(q[r0 + i, h * g:(h + 1) * g].double() @ ks.T * scale, -1)
                out[r0 + i, h * g:(h + 1) * g] = p @ vs
                size[r0 + i, h * g:(h + 1) * g] = p @ vs.abs()
    return out, size
