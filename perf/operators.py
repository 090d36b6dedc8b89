"""Cases of the paged KV cache's operators: what is measured, in plain torch and through this package.

The cache of one layer is a pool of pages [num_pages, Hkv, page, D] for the keys and one for the values; row t of
sequence b lies in page page_table[b, t // page], at row t % page. A pool holds fp16, or e4m3 with one power-of-two scale
2^e for each page and kv head (value = code * 2^e). Three operators:

  append   rotates k (and q) by rotate-half angles pos * theta^(-2i/D), pos = seq_lens[b] + i, and puts k and v into the
           pages. An e4m3 page takes the smallest e in [-15, 8] with amax <= 448 * 2^e over its new rows, or keeps the
           one that its rows before them have, if that is larger; if e grows, those rows are rounded again.
  decode   appends one token a sequence, then attends it to all keys of its sequence: softmax(q k^T / sqrt(D)) v.
  prefill  appends new tokens of every sequence, then attends each to the keys up to its own position.
"""
import math
import random

import torch

own = False

THETA = 10000.0

# ---------------------------------------------------------------- cases


def listed():
    def case(name, op, **kw):
        base = dict(cache="e4m3", head_dim=128, q_heads=32, kv_heads=32, page=16, seqs=1, cached_lo=0, cached_hi=0,
                    new_lo=1, new_hi=1)
        base.update(kw)
        return dict(name=name, op=op, **base)

    return [
        # one user's next token (7B heads): nothing but latency
        case("append_token_1", "append", cached_lo=515, cached_hi=515),
        # a full serving batch's tokens, 70B heads, every length another
        case("append_tokens_256", "append", q_heads=64, kv_heads=8, page=64, seqs=256, cached_lo=17, cached_hi=1100),
        # the prompts of the prefill benchmark: 16 of 256 to 4096 tokens, 7B heads, into an empty cache
        case("append_prompts_16", "append", page=64, seqs=16, new_lo=256, new_hi=4096),
        # chunks of prompts that begin inside a page, an unquantised cache, small heads
        case("append_chunks_fp16", "append", cache="fp16", head_dim=64, q_heads=14, kv_heads=2, page=32, seqs=5,
             cached_lo=1, cached_hi=900, new_lo=100, new_hi=777),
        # one user's decode step at 512 keys (7B heads)
        case("decode_1x512", "decode", cached_lo=512, cached_hi=512),
        # the decode benchmark: batch 32 at 4096 keys, 70B heads
        case("decode_32x4096", "decode", q_heads=64, kv_heads=8, page=64, seqs=32, cached_lo=4096, cached_hi=4096),
        # ragged batch, 7B heads, small pages: 64 sequences of 128 to 8192 keys
        case("decode_varlen_64", "decode", seqs=64, cached_lo=128, cached_hi=8192),
        # few long sequences, 70B heads
        case("decode_4x32768", "decode", q_heads=64, kv_heads=8, page=128, seqs=4, cached_lo=32768, cached_hi=32768),
        # an unquantised cache, a group of 3, odd lengths
        case("decode_ragged_fp16", "decode", cache="fp16", q_heads=24, kv_heads=8, page=32, seqs=17, cached_lo=1,
             cached_hi=5000),
        # a few proposed tokens a sequence, checked in one pass over the cache
        case("prefill_verify_8x5", "prefill", q_heads=32, kv_heads=8, page=16, seqs=8, cached_lo=900, cached_hi=3000,
             new_lo=2, new_hi=5),
        # the prefill benchmark's prompts, from an empty cache
        case("prefill_prompts_16", "prefill", page=64, seqs=16, new_lo=256, new_hi=4096),
        # a later chunk of two long prompts, 70B heads
        case("prefill_chunk_2x2048", "prefill", q_heads=64, kv_heads=8, page=64, seqs=2, cached_lo=12000,
             cached_hi=14001, new_lo=2048, new_hi=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    d = rng.choice([64, 128, 128, 256]) if op != "prefill" else 128
    kv = rng.choice([1, 2, 4, 5, 8, 32])
    group = rng.choice([1, 2, 3, 4, 7, 8] + ([16] if d < 256 else []))
    page = rng.choice([16, 32, 64] + ([128] if d < 256 else []))
    seqs = _log(rng, 1, 64)
    # a bound on the tokens of all sequences keeps a drawn case below the largest listed ones
    if op == "append":
        most = min(4096, max(1, 2_000_000 // (seqs * kv * (group + 2))))
        new_hi = 1 if rng.random() < 0.4 else _log(rng, 1, most)
        cached_hi = _log(rng, 1, 2000)
    elif op == "decode":
        new_hi = 1
        cached_hi = _log(rng, 1, min(32768, max(1, 5_000_000 // (seqs * kv))))
    else:
        new_hi = _log(rng, 1, min(2048, max(1, 1_000_000 // (seqs * kv * group))))
        cached_hi = _log(rng, 1, min(8192, max(1, 4_000_000 // (seqs * kv * group)), max(1, 40_000_000 // (seqs * kv * group * new_hi))))
    return dict(op=op, cache=rng.choice(["e4m3", "e4m3", "fp16"]), head_dim=d, q_heads=kv * group, kv_heads=kv, page=page,
                seqs=seqs, cached_lo=rng.choice([0, cached_hi // 2, cached_hi]), cached_hi=cached_hi,
                new_lo=max(1, new_hi // 3), new_hi=new_hi)


def _lengths(case):
    """(cached, new) tokens of each sequence: a function of the case alone."""
    rng = random.Random("%(op)s %(seqs)d %(cached_lo)d %(cached_hi)d %(new_lo)d %(new_hi)d" % case)
    cached = [rng.randint(case["cached_lo"], case["cached_hi"]) for _ in range(case["seqs"])]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    return cached, new


def work(case):
    cached, new = _lengths(case)
    hq, hkv, d, ps, op = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["op"]
    elt = 1 if case["cache"] == "e4m3" else 2
    tokens = sum(new)
    pages = sum((t + n - 1) // ps + 1 - (t // ps if op == "append" else 0) for t, n in zip(cached, new))
    total = tokens * 2 * hq * d * 2  # q in, and q rotated or the context out
    total += tokens * 2 * hkv * d * 2 + tokens * 2 * hkv * d * elt  # new keys and values in, their rows out
    total += pages * (4 + (2 * hkv if elt == 1 else 0))  # page table and scales
    if op == "append":
        return dict(bytes=total, flops=3 * tokens * (hq + hkv) * d)
    total += sum(cached) * 2 * hkv * d * elt  # the cached keys and values, once
    pairs = sum(n * t + n * (n + 1) // 2 for t, n in zip(cached, new))
    return dict(bytes=total, flops=4 * hq * d * pairs)


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    cached, new = _lengths(case)
    B, ps, hq, hkv, d = case["seqs"], case["page"], case["q_heads"], case["kv_heads"], case["head_dim"]
    tokens = sum(new)
    pages = [(t + n + ps - 1) // ps for t, n in zip(cached, new)]
    num, width = sum(pages) + 3, max(pages) + 1
    order = torch.randperm(num, generator=g, device=dev)
    table = torch.full((B, width), -1, dtype=torch.int32)  # entries behind a sequence's last page name no page
    at, slots = 0, order.cpu().to(torch.int32)
    for b, n in enumerate(pages):
        table[b, :n] = slots[at:at + n]
        at += n
    channel = torch.exp(0.5 * torch.randn(hkv, 1, d, generator=g, device=dev))  # keys have a few large channels
    s = dict(case=case, cached=cached, new=new, table=table.to(dev),
             lens=torch.tensor(cached, dtype=torch.int32, device=dev),
             cu=torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=dev),
             q=torch.randn(tokens, hq, d, generator=g, device=dev).half(),
             k=(torch.randn(tokens, hkv, d, generator=g, device=dev) * channel.squeeze(1)).half(),
             v=torch.randn(tokens, hkv, d, generator=g, device=dev).half(),
             out=torch.zeros(tokens, hq, d, dtype=torch.float16, device=dev), workspace=None)
    kind = torch.float8_e4m3fn if case["cache"] == "e4m3" else torch.float16
    step = max(1, (1 << 26) // (hkv * ps * d))
    for name, scale in (("k", channel), ("v", 1.0)):
        pool = torch.empty(num, hkv, ps, d, dtype=kind, device=dev)
        scales = torch.empty(num, hkv, dtype=torch.uint8, device=dev) if kind != torch.float16 else None
        for i in range(0, num, step):
            x = torch.randn(min(step, num - i), hkv, ps, d, generator=g, device=dev) * scale
            if scales is not None:
                e = _exponent(x.abs().amax((2, 3)))
                scales[i:i + step] = (e + 127).to(torch.uint8)
                x = torch.ldexp(x, -e[:, :, None, None])
            pool[i:i + step] = x.to(kind)
        s[name + "_pages"], s[name + "_scales"] = pool, None if scales is None else scales.view(torch.float8_e8m0fnu)
    if own:
        from fully_custom_cuda_inference_lamma2_b200 import attn_varlen
        s["workspace"] = attn_varlen.make_paged_workspace(B, hq, hkv, d, tokens, case["new_hi"], sum(cached) + tokens)
    return s


# ---------------------------------------------------------------- one pass


def run(s):
    if own:
        return _own(s)
    c, d = s["case"], s["case"]["head_dim"]
    seq = torch.searchsorted(s["cu"], torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32), right=True) - 1
    pos = s["lens"][seq].long() + torch.arange(seq.numel(), device="cuda") - s["cu"][seq]
    angle = pos[:, None].double() * THETA ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotated(s["q"].float(), cos, sin)
    _plain_append(s, "k", _rotated(s["k"].float(), cos, sin))
    _plain_append(s, "v", s["v"].float())
    if c["op"] == "append":
        s["out"].copy_(q)
    elif c["op"] == "decode":
        s["out"].copy_(_plain_decode(s, q))
    else:
        for b, n in enumerate(s["new"]):
            _plain_prefill(s, q, b, n)
    return _outputs(s)


def _outputs(s):
    o = dict(out=s["out"], k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["k_scales"] is not None:
        o.update(k_scales=s["k_scales"], v_scales=s["v_scales"])
    return o


def _own(s):
    from fully_custom_cuda_inference_lamma2_b200 import attn_varlen as av

    op = s["case"]["op"]
    kw = dict(k_scales=s["k_scales"], v_scales=s["v_scales"], rope_theta=THETA, workspace=s["workspace"])
    if op == "append" and s["case"]["new_hi"] == 1:  # one token a sequence: rows are sequences
        av.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], q=s["q"], q_rot_out=s["out"], **kw)
    elif op == "append":
        av.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], q=s["q"], q_rot_out=s["out"],
                        cu_seqlens_q=s["cu"], max_seqlen_q=s["case"]["new_hi"], **kw)
    elif op == "decode":
        av.paged_decode(s["q"], s["k_pages"], s["v_pages"], s["out"], s["table"], s["lens"], k_new=s["k"], v_new=s["v"], **kw)
    else:
        av.paged_prefill(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["out"], s["table"], s["lens"], s["cu"],
                         s["case"]["new_hi"], **kw)
    return _outputs(s)


# ---------------------------------------------------------------- the plain form


def _exponent(amax):
    """The smallest e in [-15, 8] with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax.float())
    return torch.where(amax > 0, e - 9 + (m > 0.875), -15).clamp(-15, 8)


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s, name, rows):
    """rows [tokens, Hkv, D] (32 bits) into the pages that they touch: [sequences, pages of each] at once."""
    ps, lens, pool = s["case"]["page"], s["lens"].long(), s[name + "_pages"]
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    first, last = lens // ps, (lens + n - 1) // ps
    # a sequence with fewer pages than another names its last one again: the same rows, written twice
    page = torch.minimum(first[:, None] + torch.arange((max(s["new"]) + ps - 2) // ps + 1, device="cuda"), last[:, None])
    pid = torch.gather(s["table"].long(), 1, page)
    at = page[:, :, None] * ps + torch.arange(ps, device="cuda")
    is_old, is_new = at < lens[:, None, None], (at >= lens[:, None, None]) & (at < (lens + n)[:, None, None])
    row = (s["cu"][:-1].long()[:, None, None] + at - lens[:, None, None]).clamp(0, rows.shape[0] - 1)
    x = rows[row].transpose(2, 3)  # [B, pages, Hkv, page, D]
    is_old, is_new = is_old[:, :, None, :, None], is_new[:, :, None, :, None]
    if s[name + "_scales"] is None:
        pool[pid] = torch.where(is_new, x.half(), pool[pid])
        return
    codes, scales = pool.view(torch.uint8), s[name + "_scales"].view(torch.uint8)
    had = codes[pid]
    e_had = scales[pid].int() - 127
    e = _exponent((x.abs() * is_new).amax((3, 4)))
    e = torch.where(is_old.any(3).squeeze(-1), torch.maximum(e, e_had), e)
    x = torch.where(is_new, x, torch.ldexp(had.view(torch.float8_e4m3fn).float(), e_had[..., None, None]))
    x = torch.ldexp(x, -e[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[pid] = torch.where(is_new | is_old, x, had)
    scales[pid] = (e + 127).to(torch.uint8)


def _gathered(s, name, pid):
    """Pages pid [..., P] of a pool in 32 bits: [..., Hkv, P * page, D]."""
    pool, scales = s[name + "_pages"], s[name + "_scales"]
    if scales is None:
        x = pool[pid].float()
    else:
        x = pool.view(torch.uint8)[pid].view(torch.float8_e4m3fn).float()
        x *= scales.view(torch.uint8)[pid].view(torch.float8_e8m0fnu).float()[..., None, None]
    return x.transpose(-4, -3).flatten(-3, -2)


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(D)) v where `seen`: q [..., Hkv, rows, D], k and v [..., Hkv, keys, D]."""
    x = (q @ k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    x = x.masked_fill_(~seen, -torch.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    return (x @ v) / x.sum(-1, keepdim=True)


def _plain_decode(s, q):
    c, n = s["case"], s["lens"].long() + 1
    used = -(-(max(s["cached"]) + 1) // c["page"])
    pid = s["table"][:, :used].clamp(min=0).long()
    seen = (torch.arange(used * c["page"], device="cuda") < n[:, None])[:, None, None]
    q = q.unflatten(1, (c["kv_heads"], -1))
    v = _gathered(s, "v", pid).masked_fill_(~seen.transpose(-1, -2), 0.0)
    return _attend(q, _gathered(s, "k", pid), v, seen).flatten(1, 2)


def _plain_prefill(s, q, b, n):
    """New tokens of sequence b: query i sees the keys up to position cached + i."""
    c, t = s["case"], s["cached"][b]
    at = sum(s["new"][:b])
    pid = s["table"][b, : -(-(t + n) // c["page"])].long()
    k, v = _gathered(s, "k", pid)[:, : t + n], _gathered(s, "v", pid)[:, : t + n]
    group = c["q_heads"] // c["kv_heads"]
    seen = torch.arange(t + n, device="cuda") <= t + torch.arange(n, device="cuda").repeat(group)[:, None]
    x = q[at: at + n].unflatten(1, (c["kv_heads"], group)).permute(1, 2, 0, 3).flatten(1, 2)  # [Hkv, G * n, D]
    x = _attend(x, k, v, seen).unflatten(1, (group, n)).permute(2, 0, 1, 3).flatten(1, 2)
    s["out"][at: at + n].copy_(x)


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    """Sequence by sequence, in 64 bits: rotation as a product of complex numbers, e4m3 by its grid of values."""
    s = prepare(case, seed)
    ps, hkv, d, group = case["page"], case["kv_heads"], case["head_dim"], case["q_heads"] // case["kv_heads"]
    pools = {x: s[x + "_pages"].double() for x in "kv"}  # codes, or the values themselves
    e8 = s["k_scales"] is not None
    scales = {x: s[x + "_scales"].double() if e8 else None for x in "kv"}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    freq = torch.exp(-math.log(THETA) * torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)

    def turned(x, pos):
        z = torch.complex(x[..., : d // 2].double(), x[..., d // 2:].double())
        z = z * torch.polar(torch.ones_like(freq), pos[:, None].double() * freq)[:, None]
        return torch.cat([z.real, z.imag], -1)

    def grid(x):  # nearest e4m3 value, ties to the even code
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(x / step) * step

    at = 0
    for b, (t, n) in enumerate(zip(s["cached"], s["new"])):
        pos = torch.arange(t, t + n, device="cuda")
        q = turned(s["q"][at: at + n], pos)
        pid = s["table"][b, : (t + n + ps - 1) // ps].long()
        for x, rows in (("k", turned(s["k"][at: at + n], pos)), ("v", s["v"][at: at + n].double())):
            j = t // ps
            mine = pools[x][pid[j:]]  # [pages, Hkv, page, D]
            if e8:
                mine = mine * scales[x][pid[j:]][:, :, None, None]
            flat = mine.transpose(1, 2).reshape(-1, hkv, d)
            off = t - j * ps
            flat[off: off + n] = rows
            if e8:
                fresh = torch.zeros_like(flat)
                fresh[off: off + n] = rows
                top = fresh.view(-1, ps, hkv, d).abs().amax((1, 3))
                two = torch.exp2(torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -15, max=2.0 ** 8))))
                if off:
                    two[0] = torch.maximum(two[0], scales[x][pid[j]])
                scaled = grid(flat.view(-1, ps, hkv, d) / two[:, None, :, None]).transpose(1, 2)
                live = torch.zeros(flat.shape[0], dtype=torch.bool, device="cuda")
                live[: off + n] = True
                pools[x][pid[j:]] = torch.where(live.view(-1, 1, ps, 1), scaled, pools[x][pid[j:]])
                scales[x][pid[j:]] = two
            else:
                pools[x][pid[j:]] = flat.view(-1, ps, hkv, d).transpose(1, 2)
        if case["op"] == "append":
            out[at: at + n] = q
        else:
            held = {}
            for x in "kv":
                y = pools[x][pid]
                y = y * scales[x][pid][:, :, None, None] if e8 else y
                held[x] = y.transpose(0, 1).reshape(hkv, -1, d)[:, : t + n]
            for i in range(0, n, 512):  # 512 queries at a time
                m = min(512, n - i)
                w = torch.einsum("nhgd,hld->hgnl", q[i: i + m].view(m, hkv, group, d), held["k"]) * d ** -0.5
                hide = torch.arange(t + n, device="cuda")[None] > pos[i: i + m, None]
                w = torch.softmax(w.masked_fill_(hide, -torch.inf), -1)
                out[at + i: at + i + m] = torch.einsum("hgnl,hld->nhgd", w, held["v"]).reshape(m, -1, d)
        at += n
    o = dict(out=out, k_pages=pools["k"], v_pages=pools["v"])
    if e8:
        o.update(k_scales=scales["k"], v_scales=scales["v"])
    return o
