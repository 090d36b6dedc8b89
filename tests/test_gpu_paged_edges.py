"""GPU checks of the paged operators at the edges of their ranges: the largest queries and keys, scale bytes that no append
makes, weights far below the largest, calls that are refused in part, bounds far above what a call holds."""
import math

import pytest
import torch

import paged_helpers as H
from helpers import randn_half
from oracle import paged_oracle as P
from test_gpu_paged import (CAPACITY, DEV, check_whole_append, exact_rotation, new_tokens, rotated_queries, run_append,
                            run_decode)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def av():
    import fully_custom_cuda_inference_lamma2_b200 as pkg

    return pkg.attn_varlen


def prefill(av, c, t, scale=None, advance=False, max_new=None, max_kv=None, d=None):
    """paged_prefill of t over c: device cache, out (7.0 where nothing was written), error word."""
    d = d or H.to_device(c)
    q, k, v = t["q"].to(DEV), t["k"].to(DEV), t["v"].to(DEV)
    out = torch.full_like(q, 7.0)
    B, hq, D = len(c["new"]), q.shape[1], q.shape[2]
    most = max_new or max(c["new"])
    kv = max_kv if max_kv is not None else sum(max(n, 0) for n in c["new"]) + int(c["T"].clamp(min=0).sum())
    ws = av.make_paged_workspace(B, hq, c["hkv"], D, q.shape[0], most, kv)
    av.paged_prefill(q, k, v, d["k"], d["v"], out, d["table"], d["T"], t["cu"].to(DEV), most, k_scales=d["k_scales"],
                     v_scales=d["v_scales"], scale=-1.0 if scale is None else scale, advance=advance, workspace=ws,
                     max_kv_tokens=kv)
    torch.cuda.synchronize()
    return d, out.cpu(), av.paged_read_error(ws)


def seq_of_rows(c):
    return [b for b, n in enumerate(c["new"]) for _ in range(n)]


# ---------------------------------------------------------------- the largest queries and keys

@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("new", [[130, 65], [10, 3]])
def test_prefill_largest_queries(av, e4m3, new):
    """Queries whose rotation passes fp16's range, in long chunks and short ones: their scores are finite."""
    c = H.make_cache([33, 200], new, 1, 128, 32, e4m3, seed=401)
    t = new_tokens(c, 2, seed=402)
    t["q"] = (torch.sign(t["q"].float()) * 65504.0).half()
    d, out, err = prefill(av, c, t, scale=1e-6)
    assert err == 0 and rotated_queries(t).abs().max() > 70000
    H.check_attention(out, rotated_queries(t), H.back(d), c["table"], [p + 1 for p in t["pos"]], seq_of_rows(c), 1e-6,
                      "largest queries", q_fp16=True)


@pytest.mark.parametrize("new", [[130, 40], [9, 3], [1, 1]])
def test_prefill_largest_keys_of_e4m3_pages(av, new):
    """Rotated keys above fp16's range, new ones and cached ones: a chunk of any length sees what the pages hold."""
    T = [100, 37]
    c = H.make_cache(T, new, 2, 128, 16, True, seed=403)
    g = torch.Generator().manual_seed(404)
    live = c["k"].view(torch.uint8) != 0x7F
    big = torch.tensor([288.0, 320.0, 352.0, -352.0, 256.0, -288.0])[torch.randint(0, 6, c["k"].shape, generator=g)]
    c["k"] = torch.where(live, big.to(H.F8).view(torch.uint8), c["k"].view(torch.uint8)).view(H.F8)
    c["k_scales"].fill_(135)
    t = new_tokens(c, 4, seed=405)
    t["k"] = (torch.sign(t["k"].float()) * 65504.0).half()
    d, out, err = prefill(av, c, t, scale=1e-6)
    assert err == 0
    after = H.back(d)
    assert float(after["k"].float().nan_to_num(0).abs().max()) * 256 > 80000
    H.check_attention(out, rotated_queries(t), after, c["table"], [p + 1 for p in t["pos"]], seq_of_rows(c), 1e-6, "largest keys",
                      q_fp16=max(new) * 2 > 64)


# ---------------------------------------------------------------- scale bytes that no append makes

@pytest.mark.parametrize("how", ["token", "rows", "decode"])
@pytest.mark.parametrize("byte", [0, 1, 3, 7, 20, 90, 111])
def test_append_to_a_page_of_a_tiny_scale(av, how, byte):
    """Rows on a page whose scale is far below the new one are rounded to zero, never to something larger."""
    T, page = [5, 20, 31], 32
    new = [1, 1, 1] if how != "rows" else [2, 5, 1]
    for factor in (3.0, 400.0, 20000.0):
        c = H.make_cache(T, new, 2, 128, page, True, seed=411)
        c["k_scales"].fill_(byte)
        c["v_scales"].fill_(byte)
        t = new_tokens(c, 2, seed=412)
        for x in "kv":
            t[x] = (t[x].float() * factor).clamp(-60000, 60000).half()
        if how == "decode":
            d, out, q_rot, err = run_decode(av, c, t)
            assert out.isfinite().all()
        else:
            d, q_rot, err = run_append(av, c, t, how == "rows")
        assert err == 0
        check_whole_append(c, t, d, q_rot, 128)


@pytest.mark.parametrize("how", ["token", "rows", "decode"])
@pytest.mark.parametrize("byte", [136, 150, 200, 253, 254])
def test_append_to_a_page_of_a_large_scale(av, how, byte):
    """A present scale above the new rows' own is kept; the rows round to it, infinities saturate."""
    T, page = [5, 20], 32
    new = [1, 1] if how != "rows" else [2, 5]
    c = H.make_cache(T, new, 1, 128, page, True, seed=413)
    c["v_scales"].fill_(byte)
    t = new_tokens(c, 2, seed=414)
    t["v"] = (t["v"].float() * 20000).clamp(-60000, 60000).half()
    first = [int(x) for x in t["cu"][:-1]]
    t["v"][first[0], 0, 3], t["v"][first[1], 0, 4] = float("inf"), float("-inf")
    d, q_rot, err = run_decode(av, c, t)[::2] + (0,) if how == "decode" else run_append(av, c, t, how == "rows")
    after = H.back(d)
    got = after["v"].view(torch.uint8)
    for b in range(2):
        p = int(c["table"][b, 0])
        assert int(after["v_scales"][p, 0]) == byte
        assert torch.equal(got[p, 0, : T[b]], c["v"].view(torch.uint8)[p, 0, : T[b]])
        for i in range(new[b]):
            x = t["v"][first[b] + i, 0].double() * 2.0 ** (127 - byte)
            want = P.e4m3_grid(x.clamp(-448, 448))
            assert torch.equal(after["v"][p, 0, T[b] + i].double(), want), (b, i)


@pytest.mark.parametrize("new", [[130, 40], [130, 0]])
def test_long_chunk_over_pages_of_a_scale_past_fp16(av, new):
    """Long chunks hold cached rows in fp16: a live page whose scale no append makes (above 2^8) is reported, and what it
    holds becomes no NaN; one that is far below holds zeros, which are exact."""
    T = [40, 37]
    c = H.make_cache(T, new, 1, 128, 16, True, seed=415)
    t = new_tokens(c, 2, seed=416)
    page = int(c["table"][0, 1])
    for byte, err_want in ((136, 16), (143, 16), (150, 16), (254, 16), (135, 0), (0, 0)):
        for name in "kv":
            e = c[name + "_scales"].clone()
            e[page, 0] = byte
            codes = c[name].view(torch.uint8).clone()
            codes[page] = 0
            cc = dict(c, **{name + "_scales": e, name: codes.view(H.F8)})
            d, out, err = prefill(av, cc, t)
            assert err == err_want, (byte, name)
            assert out.isfinite().all()
            if err == 0 or name == "v":  # zeros are zeros at any scale
                n = len(t["pos"])
                H.check_attention(out[:n], rotated_queries(t), H.back(d), c["table"], [p + 1 for p in t["pos"]], seq_of_rows(c),
                                  128 ** -0.5, f"byte {byte}", q_fp16=True)


def test_long_chunk_appends_to_a_page_of_a_scale_past_fp16(av):
    """The same for a page that gets the chunk's first rows and keeps its scale."""
    for byte, err_want in ((140, 16), (135, 0)):
        c = H.make_cache([5], [130], 1, 128, 16, True, seed=417)
        c["v"].view(torch.uint8)[int(c["table"][0, 0])] = 0
        c["v_scales"][int(c["table"][0, 0])] = byte
        d, out, err = prefill(av, c, new_tokens(c, 2, seed=418))
        assert err == err_want and out.isfinite().all()


# ---------------------------------------------------------------- weights far below the largest

@pytest.mark.parametrize("D,e4m3", [(64, False), (128, False), (256, False), (64, True), (256, True), (128, True)])
def test_decode_many_keys_far_below_one(av, D, e4m3):
    """One key of value 0 takes nearly all of every row, and what 16384 others of value 1 share (e^-gap each) is the
    result. They all lie behind it in one CTA's stretch: 600 sequences name the same pages, two units a CTA.

    A weight is off by 2^-11 of itself at most as fp16 (2^-12 as three parts), the sums by 16384 * 2^-24 and the result by
    2^-12 and 2^-25. Weights below 2^-28 of the largest need not count: gap 18 is 2^-26."""
    T, B, page = 16384, 600, 32
    for gap, lost in ((14.0, 0.0), (18.0, 0.0)):
        num = T // page
        k = torch.zeros(num, 1, page, D)
        v = torch.ones(num, 1, page, D)
        k[0, 0, 0, 0], v[0, 0, 0] = 8.0, 0.0
        kind = H.F8 if e4m3 else torch.float16
        k, v = k.to(kind).to(DEV), v.to(kind).to(DEV)
        scales = torch.full((num, 1), 127, dtype=torch.uint8, device=DEV).view(H.E8) if e4m3 else None
        table = torch.arange(num, dtype=torch.int32, device=DEV).expand(B, num).contiguous()
        lens = torch.full((B,), T, dtype=torch.int32, device=DEV)
        q = torch.zeros(B, 2, D, dtype=torch.float16, device=DEV)
        q[:, :, 0] = 8.0
        out = torch.empty_like(q)
        av.paged_decode(q, k, v, out, table, lens, k_scales=scales, v_scales=scales, scale=gap / 64.0)
        rest = (T - 1) * math.exp(-gap)
        want = rest / (1 + rest)
        tol = want * (2.0 ** -10 + 2 * T * 2.0 ** -24) + 2.0 ** -25
        worst = float((out.double() - want).abs().max())
        assert worst <= tol, f"gap {gap}: {worst / want:.3g} of the result lost"


@pytest.mark.parametrize("e4m3", [True, False])
def test_long_chunk_many_keys_far_below_one(av, e4m3):
    """The same for a chunk of 70 tokens behind them: there a weight is fp16 and the largest lies between 2^7 and 2^15, so
    that each is off by 2^-32 of the largest at most, or by 2^-11 of itself."""
    T, n, page = 16384, 70, 64
    pages = T // page + 2
    k = torch.zeros(pages, 1, page, 128)
    v = torch.ones(pages, 1, page, 128)
    k[0, 0, 0, 0], v[0, 0, 0] = 8.0, 0.0
    kind = H.F8 if e4m3 else torch.float16
    for gap in (14.0, 18.0):
        kp, vp = k.to(kind).to(DEV), v.to(kind).to(DEV)
        scales = [torch.full((pages, 1), 127, dtype=torch.uint8, device=DEV).view(H.E8) if e4m3 else None for _ in range(2)]
        table = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, pages)
        lens = torch.tensor([T], dtype=torch.int32, device=DEV)
        q = torch.zeros(n, 1, 128, dtype=torch.float16, device=DEV)
        q[:, :, 0] = 8.0
        out = torch.empty_like(q)
        av.paged_prefill(q, torch.zeros_like(q), torch.ones_like(q), kp, vp, out, table, lens,
                         torch.tensor([0, n], dtype=torch.int32, device=DEV), n, k_scales=scales[0], v_scales=scales[1],
                         scale=gap / 64.0, rotary_dim=0)
        keys = T + 1 + torch.arange(n, dtype=torch.float64)
        rest = (keys - 1) * math.exp(-gap)
        want = (rest / (1 + rest))[:, None, None]
        tol = keys[:, None, None] * 2.0 ** -32 + want * (2.0 ** -10 + 2 * T * 2.0 ** -24) + 2.0 ** -25
        worst = ((out.cpu().double() - want).abs() / tol).max()
        assert worst <= 1, f"gap {gap}: {float(worst):.3g} times the tolerance, {float(out.max() / want.max()):.3g} of the result"


@pytest.mark.parametrize("D", [128, 64, 256])
@pytest.mark.parametrize("group", [2, 16])
def test_decode_values_of_uneven_scales(av, D, group):
    """Pages whose V scales differ by 2^20, the large ones empty in half of the dims: there the small pages alone are the
    result, and they lose nothing to the large ones' weights.

    Tolerance: as in paged_helpers.check_attention, without a term that is relative to the largest weight."""
    if D == 256 and group == 16:
        group = 8
    T = [200, 333]
    c = H.make_cache(T, [0, 0], 1, D, 16, True, seed=441)
    c["new"] = [1, 1]
    c["v_scales"][:] = 127 - 12
    large = torch.arange(c["v"].shape[0]) % 2 == 0
    c["v_scales"][large] = 127 + 8
    codes = c["v"].view(torch.uint8)
    codes[large, :, :, D // 2:] = 0
    t = new_tokens(c, group, seed=442)
    d, out, q_rot, err = run_decode(av, c, t, append=False, scale=0.02)
    assert err == 0
    for b in range(2):
        k, v = P.keys_values(c["k"], c["v"], c["k_scales"], c["v_scales"], c["table"][b], T[b], 0)
        for h in range(group):
            o, w, s, _ = P.attention(t["q"][b, h].double(), k, v, 0.02)
            eps = 2 * s * (2.0 ** -12 + 2.0 ** -16 + 2.0 ** -20)
            tol = w * (eps + 2.0 ** -11 + 2.0 ** -19 + 2 * T[b] * 2.0 ** -24) + o.abs() * 2.0 ** -11 + 2.0 ** -25
            worst = ((out[b, h].double() - o).abs() / tol)[D // 2:].max()
            assert worst <= 1, f"sequence {b}, row {h}: {float(worst):.3g} times the tolerance"


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("byte", [0, 10, 100, 127])
def test_decode_over_a_zeroed_cache(av, D, byte):
    """Codes and scale bytes of a cache that was zeroed, also where a sequence is cut over many CTAs: zeros."""
    T = [5000, 1, 0, 300]
    c = H.make_cache(T, [1] * 4, 1, D, 16, True, seed=443, poison=False)
    for name in "kv":
        c[name].view(torch.uint8).zero_()
        c[name + "_scales"].fill_(byte)
    d, out, q_rot, err = run_decode(av, c, new_tokens(c, 4, seed=444), append=False)
    assert err == 0 and (out == 0).all()
    # a row of ones at the end of each
    t = new_tokens(c, 4, seed=445)
    t["v"].fill_(1.0)
    d, out, q_rot, err = run_decode(av, c, t, scale=1e-9)
    n = torch.tensor(T).double()[:, None, None] + 1  # scores of 1e-9 * 128 at most: equal weights, 1 / n in each dim
    assert err == 0 and ((out.double() * n - 1).abs() <= 2.0 ** -10 + 5001 * 2.0 ** -24 + n * 2.0 ** -25).all()


# ---------------------------------------------------------------- calls that are refused in part

def test_long_chunk_without_room_leaves_its_pages(av):
    """A sequence whose expanded keys have no room is not served: its pages, scales, rows of out and length stay."""
    T, new = [20, 30, 10], [70, 100, 66]
    c = H.make_cache(T, new, 2, 128, 16, True, seed=421)
    t = new_tokens(c, 4, seed=422)
    for name in "kv":
        t[name] = (t[name].float() * 100).clamp(-60000, 60000).half()  # would grow the scale of the page that holds row T
    # the first and the third fit, the second does not
    d, out, err = prefill(av, c, t, advance=True, max_kv=20 + 70 + 10 + 66 + 20)
    assert err == CAPACITY and d["T"].cpu().tolist() == [90, 30, 76]
    after = H.back(d)
    mine = c["table"][1][c["table"][1] >= 0].long()
    for name in "kv":
        assert torch.equal(after[name].view(torch.uint8)[mine], c[name].view(torch.uint8)[mine]), "pages of the refused sequence"
        assert torch.equal(after[name + "_scales"][mine], c[name + "_scales"][mine]), "scales of the refused sequence"
    rows = list(range(70)) + list(range(170, 236))
    assert (out[70:170] == 7.0).all()
    pos = [t["pos"][r] for r in rows]
    H.check_attention(out[rows], exact_rotation(t["q"][rows], pos, 128), after, c["table"], [p + 1 for p in pos],
                      [0] * 70 + [2] * 66, 128 ** -0.5, "others", q_fp16=True)


def test_long_chunk_of_offsets_that_share_rows(av):
    """Offsets that run backwards, so that more work is asked for than the rows of the call allow: nothing is served, and
    lengths, pages and scales stay."""
    n, B = 2560, 5
    c = H.make_cache([3] * B, [n, 0, n, 0, n], 1, 128, 128, True, seed=423)
    c["new"] = [n, 0, 0, 0, 0]
    t = new_tokens(c, 2, seed=424)
    t["cu"] = torch.tensor([0, n, 0, n, 0, n], dtype=torch.int32)
    d, out, err = prefill(av, c, t, advance=True, max_new=n, max_kv=3 * (n + 3))
    assert err == CAPACITY and d["T"].cpu().tolist() == [3] * B and (out == 7.0).all()
    after = H.back(d)
    for name in "kv":
        assert torch.equal(after[name].view(torch.uint8), c[name].view(torch.uint8))
        assert torch.equal(after[name + "_scales"], c[name + "_scales"])


@pytest.mark.parametrize("D,e4m3", [(128, True), (64, True), (128, False)])
def test_lengths_past_what_a_line_holds(av, D, e4m3):
    """Sequences of 2^30 rows are more tiles than the line's numbers hold: the call is reported, and neither the lengths nor
    out nor the pages change. (No page of them is looked up.)"""
    page, pages = 16, 1 << 26
    B, hkv = 2, 2
    kind = H.F8 if e4m3 else torch.float16
    pool = torch.zeros(4, hkv, page, D, dtype=torch.uint8 if e4m3 else torch.float16, device=DEV)
    scales = torch.full((4, hkv), 127, dtype=torch.uint8, device=DEV).view(H.E8) if e4m3 else None
    table = torch.full((B, pages), -1, dtype=torch.int32, device=DEV)
    lens = torch.full((B,), 1 << 29, dtype=torch.int32, device=DEV)
    q, k = randn_half((B, 4, D), 425).to(DEV), randn_half((B, hkv, D), 426).to(DEV)
    out = torch.full_like(q, 7.0)
    ws = av.make_paged_workspace(B, 4, hkv, D, B)
    before = pool.clone()
    av.paged_decode(q, pool.view(kind), pool.view(kind), out, table, lens, k_scales=scales, v_scales=scales, k_new=k, v_new=k,
                    advance=True, workspace=ws)
    torch.cuda.synchronize()
    assert av.paged_read_error(ws) == CAPACITY
    assert lens.tolist() == [1 << 29] * B and (out == 7.0).all() and torch.equal(pool, before)


@pytest.mark.parametrize("e4m3", [True, False])
def test_append_to_lengths_that_are_none(av, e4m3):
    """Negative lengths and ones past the table, ragged rows: reported, nothing of theirs is written."""
    T, new = [20, 17, 40, 0], [5, 70, 3, 33]
    c = H.make_cache(T, new, 2, 128, 16, e4m3, seed=433)
    t = new_tokens(c, 2, seed=434)
    room = c["table"].shape[1] * 16
    for bad in (-1, -5, -100, -2 ** 31, room - 69, 2 ** 31 - 1):
        cc = dict(c, T=torch.tensor([20, bad, 40, 0], dtype=torch.int32))
        d, q_rot, err = run_append(av, cc, t, True, advance=True)
        assert err == CAPACITY and d["T"].cpu().tolist() == [25, bad, 43, 33]
        after = H.back(d)
        mine = c["table"][1][c["table"][1] >= 0].long()
        for name in "kv":
            assert torch.equal(H.bits(after[name])[mine], H.bits(c[name])[mine])
        assert (q_rot[5:75] == 7.0).all()


def test_short_chunks_of_too_many_sequences(av):
    """A call that is refused leaves the pages alone: the check comes before the append."""
    B = 20000
    pool = torch.zeros(B, 1, 16, 128, dtype=torch.uint8, device=DEV)
    scales = torch.full((B, 1), 120, dtype=torch.uint8, device=DEV)
    table = torch.arange(B, dtype=torch.int32, device=DEV).view(B, 1)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    q = randn_half((B, 1, 128), 435).to(DEV)
    out = torch.full_like(q, 7.0)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    before = av.launch_count()
    with pytest.raises(RuntimeError, match="batch too large"):
        av.paged_prefill(q, q, q, pool.view(H.F8), pool.view(H.F8), out, table, lens, cu, 1, k_scales=scales, v_scales=scales, advance=True)
    torch.cuda.synchronize()
    assert av.launch_count() == before
    assert (pool == 0).all() and (scales == 120).all() and (lens == 0).all() and (out == 7.0).all()


# ---------------------------------------------------------------- bounds far above what a call holds

@pytest.mark.parametrize("e4m3", [True, False])
def test_append_under_a_bound_of_any_size(av, e4m3):
    """max_seqlen_q is a bound: what a call holds decides its work, whatever the bound says."""
    T, new = [5, 0, 63, 1000], [40, 1, 0, 130]
    c = H.make_cache(T, new, 2, 128, 16, e4m3, seed=431)
    t = new_tokens(c, 4, seed=432)
    seen = []
    for bound in (130, 1 << 20, 2 ** 31 - 1):
        d = H.to_device(c)
        q_rot = torch.full_like(t["q"], 7.0).to(DEV)
        av.paged_append(t["k"].to(DEV), t["v"].to(DEV), d["k"], d["v"], d["table"], d["T"], k_scales=d["k_scales"],
                        v_scales=d["v_scales"], q=t["q"].to(DEV), q_rot_out=q_rot, cu_seqlens_q=t["cu"].to(DEV), max_seqlen_q=bound)
        torch.cuda.synchronize()
        check_whole_append(c, t, d, q_rot.cpu(), 128)
        seen.append((H.bits(H.back(d)["k"]), H.bits(H.back(d)["v"])))
    for a, b in seen[1:]:
        assert torch.equal(a, seen[0][0]) and torch.equal(b, seen[0][1])


@pytest.mark.parametrize("how,e4m3,D", [("append", False, 64), ("append", True, 128), ("append", True, 256),
                                        ("prefill", False, 128), ("prefill", True, 128)])
def test_append_of_many_pages_by_few_blocks(av, how, e4m3, D):
    """One long run of tokens beside thousands of short ones, under a bound that any could reach: every page of each is
    written. (The values are exact in e4m3 at any scale of theirs.)"""
    B = 3000
    T = [(7 * b) % 33 for b in range(B)]
    new = [1 + b % 3 for b in range(B)]
    new[1234] = 5000
    page = 16
    cu = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32)
    need = torch.tensor([-(-(a + n) // page) for a, n in zip(T, new)])
    table = torch.full((B, int(need.max())), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, : need[b]] = torch.arange(at, at + int(need[b]), dtype=torch.int32)
        at += int(need[b])
    kind = H.F8 if e4m3 else torch.float16
    pools = [torch.zeros(at, 1, page, D, dtype=torch.float16, device=DEV).to(kind) for _ in range(2)]
    scales = [torch.full((at, 1), 112, dtype=torch.uint8, device=DEV).view(H.E8) if e4m3 else None for _ in range(2)]
    n = int(cu[-1])
    v = ((torch.arange(n * D) * 5 // 3) % 8 + 8).view(n, 1, D).half().to(DEV)
    lens = torch.tensor(T, dtype=torch.int32, device=DEV)
    kw = dict(k_scales=scales[0], v_scales=scales[1], rotary_dim=0, advance=True)
    if how == "append":
        av.paged_append(v, v, *pools, table.to(DEV), lens, cu_seqlens_q=cu.to(DEV), max_seqlen_q=1 << 30, **kw)
    else:
        out = torch.zeros_like(v)
        av.paged_prefill(v, v, v, *pools, out, table.to(DEV), lens, cu.to(DEV), 1 << 30, max_kv_tokens=n + sum(T), **kw)
        assert out.isfinite().all() and (out >= 0).all() and (out <= 15).all() and (out[cu[:-1].long()][:1] > 0).all()
    assert lens.tolist() == [a + b for a, b in zip(T, new)]
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new))
    pos = torch.tensor(T)[seq] + torch.arange(n) - cu[:-1].long()[seq]
    page_of = table[seq, pos // page].long()
    for x, s in zip(pools, scales):
        x = x.float().cpu() * (s.float().cpu()[:, :, None, None] if e4m3 else 1.0)
        assert torch.equal(x[page_of, 0, pos % page], v.float().cpu()[:, 0])
        assert int((x != 0).sum()) == n * D
