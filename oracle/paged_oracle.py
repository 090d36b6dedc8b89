"""CPU oracle of the paged KV cache's operators, in 64 bits — TEST INFRASTRUCTURE ONLY.

One sequence and one row at a time, from the definitions in include/fcci_paged.h:

  rope           rotate-half at position pos, angles pos * theta^(-2j / rotary_dim)
  scale_exponent the smallest e in [-15, 8] with amax <= 448 * 2^e
  e4m3_grid      the nearest e4m3 value (ties to even, saturating at 448)
  append         the pools after an append, and the exact rotated rows
  attention      softmax(q k^T scale) v over what the pools hold

The pools are the caller's tensors on the CPU: fp16, or float8_e4m3fn with uint8 scales.
"""
from __future__ import annotations

import math

import torch


def rope(x: torch.Tensor, pos: int, rotary_dim: int, theta: float) -> torch.Tensor:
    """x [..., D] rotated at position pos, float64."""
    x = x.double().clone()
    half = rotary_dim // 2
    if half == 0:
        return x
    ang = torch.tensor([math.fmod(pos * theta ** (-2.0 * j / rotary_dim), 2 * math.pi) for j in range(half)],
                       dtype=torch.float64)
    a, b = x[..., :half].clone(), x[..., half:rotary_dim].clone()
    x[..., :half] = a * ang.cos() - b * ang.sin()
    x[..., half:rotary_dim] = b * ang.cos() + a * ang.sin()
    return x


def scale_exponent(amax: float) -> int:
    for e in range(-15, 8):
        if amax <= 448.0 * 2.0 ** e:
            return e
    return 8


def e4m3_grid(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of each float64 x (three mantissa bits, exponent at least -6)."""
    mag = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(mag.clamp(min=2.0 ** -6))) - 3)
    return torch.where(x.isnan(), x, torch.sign(x) * torch.round(mag / step) * step)


def values(pool: torch.Tensor, scales, page: int, h: int) -> torch.Tensor:
    """What page `page` of kv head h holds: [page_size, D] float64."""
    v = pool[page, h].double()
    return v if scales is None else v * 2.0 ** (int(scales[page, h]) - 127)


def append(pool, scales, table, T, cu, rows):
    """rows [tokens, Hkv, D] (float64, rotated already) into clones of pool and scales.

    Returns (values float64 [pages, Hkv, page, D] with NaN where nothing was appended or
    re-rounded, exponents {(page, h): e}): what the appended rows must come to."""
    ps, hkv = pool.shape[2], pool.shape[1]
    want = torch.full(pool.shape, float("nan"), dtype=torch.float64)
    exps = {}
    for b in range(len(T)):
        t, n = int(T[b]), int(cu[b + 1] - cu[b])
        if n == 0:
            continue
        for j in range(t // ps, (t + n - 1) // ps + 1):
            page = int(table[b, j])
            lo, hi = max(t, j * ps), min(t + n, (j + 1) * ps)
            mine = rows[int(cu[b]) + lo - t: int(cu[b]) + hi - t]
            for h in range(hkv):
                if scales is None:
                    want[page, h, lo - j * ps: hi - j * ps] = mine[:, h]
                    continue
                finite = mine[:, h][~mine[:, h].isnan()].abs()
                e = scale_exponent(float(finite.max()) if finite.numel() else 0.0)
                if lo > j * ps:
                    had = int(scales[page, h]) - 127
                    if had >= e:
                        e = had
                    else:
                        old = values(pool, scales, page, h)[: lo - j * ps]
                        want[page, h, : lo - j * ps] = e4m3_grid(old * 2.0 ** -e) * 2.0 ** e
                exps[(page, h)] = e
                want[page, h, lo - j * ps: hi - j * ps] = mine[:, h]
    return want, exps


def keys_values(k_pool, v_pool, k_scales, v_scales, table_row, length, h):
    """The first `length` rows of a sequence, kv head h: two [length, D] float64."""
    ps = k_pool.shape[2]
    pages = [int(x) for x in table_row[: -(-length // ps)]]
    k = [values(k_pool, k_scales, p, h) for p in pages]
    v = [values(v_pool, v_scales, p, h) for p in pages]
    if not pages:
        z = torch.zeros(0, k_pool.shape[3], dtype=torch.float64)
        return z, z
    return torch.cat(k)[:length], torch.cat(v)[:length]


def attention(q, k, v, scale):
    """(out [D], weights @ |v| [D], largest sum|q k| scale, largest weight) of one query row in float64."""
    if k.shape[0] == 0:
        z = torch.zeros(q.shape[-1], dtype=torch.float64)
        return z, z, 0.0, 0.0
    x = (k @ q.double()) * scale
    p = torch.softmax(x, 0)
    return p @ v, p @ v.abs(), float(((k.abs() @ q.double().abs()) * scale).max()), float(p.max())
