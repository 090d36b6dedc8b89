"""How far an attention call's whole result may be from 64 bits, in the 2-norm, and the kernels' arithmetic on the CPU.

The elementwise bounds of paged_helpers.check_attention add up what each rounding may do at worst. Roundings are as good as
independent, so a whole call is far closer, and a part that is missing shows in its 2-norm. Each of these is the root mean
square of an error spread evenly over a rounding's step, at most 2^-11 / sqrt(3) = 2.82e-4 relative to a value of the
smallest mantissa:

  the result, fp16                          2.82e-4
  the weights, fp16 (in any number of exact 8-bit parts)   2.82e-4, if one weight has it all; divided by the root of
                                            the number of keys that count otherwise
  the queries: three e4m3 parts 2^-13 / sqrt(3), two fp16 parts 2^-22, one fp16 part 2^-12 / sqrt(3) (all 2^-12 at most),
                                            times the 2-norm of the products q_i k_i in a score

SPLIT bounds the first two and a score error of as much (sqrt(3) * 2.82e-4); LONG is what the library asks of its prefill.
"""
from __future__ import annotations

import torch

import paged_helpers as H
from oracle import paged_oracle as P

SPLIT, LONG = 5e-4, 1e-3
WIDE = 0.5  # a scale under which the roundings of queries of head_dim 128 count more than the result's own


def plain_cache(T, hkv, D, page, e4m3, seed, spare_rows=1):
    """A cache (as paged_helpers.make_cache makes it) whose keys and values are N(0, 1): many keys count in each row."""
    c = H.make_cache(T, [spare_rows] * len(T), hkv, D, page, e4m3, seed=seed, poison=False)
    g = torch.Generator().manual_seed(seed + 1)
    for name in ("k", "v"):
        x = torch.randn(c[name].shape, generator=g)
        if e4m3:
            c[name + "_scales"].fill_(127 - 6)  # 448 / 64 = 7: none is cut
            c[name] = (x * 64).clamp(-448, 448).to(H.F8)
        else:
            c[name] = x.half()
    return c


def exact(q, cache, table, lens_of_row, seq_of_row, scale):
    """[rows, Hq, D] float64: attention of every row in 64 bits over what the pools hold."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    hkv = cache["k"].shape[1]
    group = q.shape[1] // hkv
    for h in range(hkv):
        held = {}
        for r in range(q.shape[0]):
            b, L = int(seq_of_row[r]), int(lens_of_row[r])
            if b not in held:
                top = max(int(n) for n, s in zip(lens_of_row, seq_of_row) if int(s) == b)
                held[b] = P.keys_values(cache["k"], cache["v"], cache["k_scales"], cache["v_scales"], table[b], top, h)
            if L:
                k, v = held[b][0][:L], held[b][1][:L]
                w = torch.softmax(q[r, h * group: (h + 1) * group].double() @ k.T * scale, -1)
                out[r, h * group: (h + 1) * group] = w @ v
    return out


def off(out, want):
    """Relative distance in the 2-norm."""
    return float((out.double() - want).norm() / want.norm())


# ---------------------------------------------------------------- the kernels' arithmetic, part by part

def e4m3_parts(x, parts):
    """x [..., D] as `parts` e4m3 values, each the rounding of what the ones before left, times 16, under one power of two."""
    up = torch.exp2(torch.floor(torch.log2(448 / x.abs().amax(-1, keepdim=True))))
    rest, total, f = x * up, torch.zeros_like(x), 1.0
    for _ in range(parts):
        p = P.e4m3_grid(rest)
        total = total + p * f
        rest, f = (rest - p) * 16, f / 16
    return total / up


def e5m2_parts(w, parts):
    """fp16 of w (at most 2^15.75) as `parts` e5m2 values, each cut off from 8 times what the ones before left."""
    rest, total, f = w.half(), torch.zeros_like(w), 1.0
    for _ in range(parts):
        p = (rest.view(torch.int16) & -256).view(torch.float16)
        total = total + p.double() * f
        rest, f = (rest - p) * 8, f / 8
    return total


def emulated(q, cache, table, lens, scale, kind, query_parts, weight_parts=4):
    """One token a sequence through the split kernels' roundings: kind "e4m3" (tensor memory) or "fp16"."""
    out = torch.zeros(q.shape, dtype=torch.float16)
    hkv = cache["k"].shape[1]
    group = q.shape[1] // hkv
    for b in range(q.shape[0]):
        for h in range(hkv):
            k, v = P.keys_values(cache["k"], cache["v"], cache["k_scales"], cache["v_scales"], table[b], int(lens[b]), h)
            x = q[b, h * group: (h + 1) * group].double()
            if kind == "e4m3":
                x = e4m3_parts(x, query_parts)
            else:
                hi = x.half().double()
                x = hi + ((x - hi).half().double() if query_parts > 1 else 0)
            s = x @ k.T * scale
            w = torch.exp(s - s.amax(-1, keepdim=True))
            held = e5m2_parts(w * 2.0 ** 13, weight_parts) / 2.0 ** 13 if kind == "e4m3" else (w * 2.0 ** 14).half().double() / 2.0 ** 14
            out[b, h * group: (h + 1) * group] = ((held @ v) / w.sum(-1, keepdim=True)).half()
    return out
