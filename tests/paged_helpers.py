"""Seeded paged caches for the tests, and the comparisons with the 64-bit oracle."""
from __future__ import annotations

import torch

from oracle import paged_oracle as P

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def make_cache(T, new, hkv, D, page, e4m3, seed, spare=3, layout="hnd", poison=True):
    """A pool whose sequences hold T[b] rows and have pages for new[b] more, in shuffled order.

    Rows that belong to nobody hold NaN (poison). layout "nhd": pages [num, page, Hkv, D] in memory;
    "sliced": a view into a wider pool."""
    g = torch.Generator().manual_seed(seed)
    B = len(T)
    need = [-(-(t + n) // page) for t, n in zip(T, new)]
    num, width = sum(need) + spare, max(need + [1]) + 1
    perm = torch.randperm(num, generator=g).tolist()
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = torch.tensor(perm[at:at + need[b]], dtype=torch.int32)
        at += need[b]
    c = dict(T=torch.tensor(T, dtype=torch.int32), new=list(new), table=table, page=page, D=D, hkv=hkv)
    for name in ("k", "v"):
        x = torch.randn(num, hkv, page, D, generator=g) * torch.exp(torch.randn(num, hkv, 1, 1, generator=g))
        live = torch.zeros(num, page, dtype=torch.bool)
        for b in range(B):
            for j in range(need[b]):
                live[int(table[b, j]), : max(0, min(page, T[b] - j * page))] = True
        scales = None
        if e4m3:
            e = torch.tensor([[P.scale_exponent(float(x[i, h].abs().max())) for h in range(hkv)] for i in range(num)])
            # pages without a live row hold an arbitrary scale byte: an append must not take it for theirs
            e = torch.where(live.any(1)[:, None], e, torch.randint(-15, 9, e.shape, generator=g))
            pool = torch.ldexp(x, -e[:, :, None, None]).clamp(-448, 448).to(F8)
            scales = (e + 127).to(torch.uint8)
            if poison:
                pool.view(torch.uint8).masked_fill_(~live[:, None, :, None], 0x7F)
        else:
            pool = x.half()
            if poison:
                pool.masked_fill_(~live[:, None, :, None], float("nan"))
        c[name], c[name + "_scales"] = pool, scales
    c["layout"] = layout
    return c


def to_device(c, dev="cuda"):
    """Device copies: pools in the cache's memory layout, tables and lengths."""
    d = {}
    for name in ("k", "v"):
        raw = c[name].view(torch.uint8) if c[name].dtype == F8 else c[name]
        raw = raw.to(dev)
        if c["layout"] == "nhd":
            raw = raw.transpose(1, 2).contiguous().transpose(1, 2)
        elif c["layout"] == "sliced":
            wide = torch.empty(raw.shape[0], raw.shape[1] + 1, raw.shape[2], raw.shape[3] + 16, dtype=raw.dtype, device=dev)
            wide.view(torch.uint8).fill_(0x7F)
            wide[:, 1:, :, 16:] = raw
            raw = wide[:, 1:, :, 16:]
        d[name] = raw.view(F8) if c[name].dtype == F8 else raw
        s = c[name + "_scales"]
        d[name + "_scales"] = None if s is None else s.to(dev).view(E8)
    d["table"], d["T"] = c["table"].to(dev), c["T"].to(dev)
    return d


def back(d):
    """The pools and scales on the CPU again."""
    out = {}
    for name in ("k", "v"):
        raw = d[name].view(torch.uint8) if d[name].dtype == F8 else d[name]
        raw = raw.cpu().contiguous()
        out[name] = raw.view(F8) if d[name].dtype == F8 else raw
        s = d[name + "_scales"]
        out[name + "_scales"] = None if s is None else s.view(torch.uint8).cpu()
    return out


def bits(t):
    return t.view(torch.uint8) if t.dtype == F8 else t.view(torch.int16)


def check_append(before, after, name, T, cu, table, exact_rows, turned):
    """The pools after an append. exact_rows [tokens, Hkv, D] float64, rotated in 64 bits.

    A stored value is the fp32 rotation, rounded once. The fp32 rotation is off by at most
    delta = 2^-21 (|x1| + |x2|): two products and a sum (3 * 2^-24), cos and sin (1.2e-7 each of angle and function).
    Rounding adds half a step: e4m3 2^-4 of the value or 2^-10 of the scale below its normals, fp16 2^-11 or 2^-25.
    Values that are not rotated are exact before the rounding, so theirs is the only right code."""
    pool, scales = after[name], after[name + "_scales"]
    want, exps = P.append(before[name], before[name + "_scales"], table, T, cu, exact_rows)
    touched = ~want.isnan()
    ps = pool.shape[2]
    # what the append does not name stays as it was, bit for bit
    new = torch.zeros(pool.shape[0], ps, dtype=torch.bool)
    for b in range(len(T)):
        for t in range(int(T[b]), int(T[b]) + int(cu[b + 1] - cu[b])):
            new[int(table[b, t // ps]), t % ps] = True
    same = bits(pool) == bits(before[name])
    assert (same | touched | new[:, None, :, None]).all(), f"{name}: a row outside the append changed"
    if scales is not None:
        expect = before[name + "_scales"].clone().int() - 127
        for (p, h), e in exps.items():
            expect[p, h] = e
        assert torch.equal(scales.int() - 127, expect), f"{name}: scale exponents"
        val = pool.double() * torch.exp2(scales.double() - 127)[:, :, None, None]
        half = torch.maximum(want.abs() * 2.0 ** -4, torch.exp2(scales.double() - 127 - 10)[:, :, None, None].expand_as(want))
    else:
        val = pool.double()
        half = torch.maximum(want.abs() * 2.0 ** -11, torch.tensor(2.0 ** -25, dtype=torch.float64))
    if turned:
        big = float(exact_rows.nan_to_num(0, 0, 0).abs().max()) * 2
        ok = (val - want).abs() <= half + 2.0 ** -21 * big
    else:
        rounded = P.e4m3_grid(want / torch.exp2(scales.double() - 127)[:, :, None, None]) * \
            torch.exp2(scales.double() - 127)[:, :, None, None] if scales is not None else want
        ok = val == rounded
    bad = touched & ~ok
    assert not bad.any(), f"{name}: {int(bad.sum())} values off, first {bad.nonzero()[0].tolist()}: " \
        f"{val[bad][0]} for {want[bad][0]}"


def check_q_rot(q_rot, exact):
    tol = exact.abs() * 2.0 ** -11 + 2.0 ** -25 + 2.0 ** -20 * exact.abs().max()
    assert ((q_rot.double() - exact).abs() <= tol).all(), float((q_rot.double() - exact).abs().max())


def check_attention(out, q, cache, table, lens_of_row, seq_of_row, scale, what="", q_fp16=False):
    """out [rows, Hq, D] against 64 bits over what the pools hold, elementwise.

    q [rows, Hq, D]: the queries rotated in 64 bits. The kernels rotate them in fp32 (off by 2^-21 of the pair's sizes)
    and hold them in two fp16 parts (2^-22), in three e4m3 parts (each at most 2^-4 of what the one before left: 2^-12;
    below 2^-10 / 256 of 448 nothing: 2^-26 of the row's largest element, which times sum|k| is at most 2^6 sum|q k|
    for the inputs here), or, with q_fp16, in one (2^-11). A score is then off by at most
    eps = (2^-12 + 2^-16 + 2^-20) * sum|q k| scale (256 fp32 products summed in any order: 256 * 2^-24), with q_fp16 by
    2^-11 of that sum, so a normalised weight by 2 eps of itself. A weight is rounded to fp16 (2^-11, or 2^-25 absolute
    below its normals), to three e4m3 parts after it (2^-12, or 2^-24 of the largest weight) and comes from an
    approximate power of two (2^-21 and less); the fp32 sums over L keys are off by L * 2^-24, above and below the
    fraction line; the result is rounded to fp16 (2^-11, or 2^-25 absolute). All of it moves out by at most that
    share of sum(weight |v|); the largest weight is at most the sum of the weights."""
    hq, D = out.shape[1], out.shape[2]
    hkv = cache["k"].shape[1]
    worst = 0.0
    for h in range(hkv):
        held = {}
        for r in range(out.shape[0]):
            b, L = int(seq_of_row[r]), int(lens_of_row[r])
            if b not in held:
                top = max(int(lens_of_row[i]) for i in range(out.shape[0]) if int(seq_of_row[i]) == b)
                held[b] = P.keys_values(cache["k"], cache["v"], cache["k_scales"], cache["v_scales"], table[b], top, h)
            k, v = held[b][0][:L], held[b][1][:L]
            for g in range(hq // hkv):
                o, w, s, top = P.attention(q[r, h * (hq // hkv) + g], k, v, scale)
                got = out[r, h * (hq // hkv) + g].double()
                vmax = v.abs().max(0).values if L else torch.zeros(D, dtype=torch.float64)
                s *= 2.0 ** -16 + (2.0 ** -11 if q_fp16 else 2.0 ** -12 + 2.0 ** -20)
                tol = w * (2 * s + 2.0 ** -11 + 2.0 ** -12 + 2.0 ** -19 + 2 * L * 2.0 ** -24) + L * 2.0 ** -24 * top * vmax \
                    + o.abs() * 2.0 ** -11 + 2.0 ** -25
                worst = max(worst, float(((got - o).abs() / tol).nan_to_num(1e9).max()))
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"
    return worst
