"""GPU parity of the paged KV cache's operators against the 64-bit oracle: append, decode, prefill."""
import math

import pytest
import torch

import paged_helpers as H
from helpers import randn_half
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
CAPACITY, PAGE_ERR = 1, 8


@pytest.fixture(scope="module")
def av():
    import fully_custom_cuda_inference_lamma2_b200 as pkg

    return pkg.attn_varlen


def new_tokens(c, hq, seed, gap=0, scale=1.0):
    """q, k, v of the new tokens (gap rows behind the last sequence), cu_seqlens, positions."""
    cu = [0]
    for n in c["new"]:
        cu.append(cu[-1] + n)
    rows = cu[-1] + gap
    pos = [int(c["T"][b]) + i for b, n in enumerate(c["new"]) for i in range(n)]
    return dict(q=randn_half((rows, hq, c["D"]), seed), k=(randn_half((rows, c["hkv"], c["D"]), seed + 1).float() * scale).half(),
                v=randn_half((rows, c["hkv"], c["D"]), seed + 2), cu=torch.tensor(cu, dtype=torch.int32), pos=pos)


def exact_rotation(x, pos, rot, theta=10000.0):
    return torch.stack([P.rope(x[i], p, rot, theta) for i, p in enumerate(pos)]) if pos else x[:0].double()


def rotated_queries(t, rot=None):
    return exact_rotation(t["q"][: len(t["pos"])], t["pos"], t["q"].shape[2] if rot is None else rot)


def run_append(av, c, t, varlen, rot=-1, theta=10000.0, advance=False, with_q=True, ws=None):
    d = H.to_device(c)
    q, k, v = t["q"].to(DEV), t["k"].to(DEV), t["v"].to(DEV)
    q_rot = torch.full_like(q, 7.0).contiguous()
    B, hq = len(c["new"]), q.shape[1]
    own_ws = ws is None
    if own_ws:
        ws = av.make_paged_workspace(B, hq, c["hkv"], c["D"], q.shape[0], max(c["new"] + [1]))
    kw = dict(cu_seqlens_q=t["cu"].to(DEV), max_seqlen_q=max(c["new"])) if varlen else {}
    av.paged_append(k, v, d["k"], d["v"], d["table"], d["T"], k_scales=d["k_scales"], v_scales=d["v_scales"],
                    q=q if with_q else None, q_rot_out=q_rot if with_q else None, rope_theta=theta, rotary_dim=rot,
                    advance=advance, workspace=ws, **kw)
    torch.cuda.synchronize()
    err = av.paged_read_error(ws)
    return d, q_rot.cpu(), err


def check_whole_append(c, t, d, q_rot, rot, theta=10000.0):
    n = len(t["pos"])
    after = H.back(d)
    k_exact = exact_rotation(t["k"][:n], t["pos"], rot, theta)
    H.check_append(c, after, "k", c["T"], t["cu"], c["table"], k_exact, rot > 0)
    H.check_append(c, after, "v", c["T"], t["cu"], c["table"], t["v"][:n].double(), False)
    H.check_q_rot(q_rot[:n], exact_rotation(t["q"][:n], t["pos"], rot, theta))
    assert (q_rot[n:] == 7.0).all(), "rows behind the last sequence were written"


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("D,page,hkv,hq,layout", [
    (128, 16, 8, 8, "hnd"), (128, 64, 2, 10, "nhd"), (64, 128, 1, 16, "sliced"), (256, 32, 3, 6, "hnd"),
    (128, 128, 1, 1, "nhd"), (64, 16, 5, 5, "hnd"), (256, 64, 1, 2, "sliced")])
def test_append_one_token(av, e4m3, D, page, hkv, hq, layout):
    T = [0, 1, page - 1, page, page + 1, 3 * page - 1, 517]
    c = H.make_cache(T, [1] * len(T), hkv, D, page, e4m3, seed=D + page, layout=layout)
    t = new_tokens(c, hq, seed=3, scale=1.7)
    d, q_rot, err = run_append(av, c, t, varlen=False)
    assert err == 0
    check_whole_append(c, t, d, q_rot, D)
    assert d["T"].cpu().tolist() == T


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("D,page,hkv,hq,layout", [
    (128, 16, 4, 8, "hnd"), (128, 64, 2, 6, "nhd"), (64, 128, 3, 3, "sliced"), (256, 64, 1, 4, "hnd"),
    (64, 16, 2, 14, "nhd"), (128, 128, 1, 9, "hnd"), (256, 16, 2, 2, "sliced")])
def test_append_prompts(av, e4m3, D, page, hkv, hq, layout):
    T = [0, 5, page - 1, page, 0, 2 * page + 3, 40]
    new = [3 * page + 1, 1, 2, page, 0, page - 3, 200]
    c = H.make_cache(T, new, hkv, D, page, e4m3, seed=D + page + 1, layout=layout)
    t = new_tokens(c, hq, seed=5, gap=3)
    d, q_rot, err = run_append(av, c, t, varlen=True, advance=True)
    assert err == 0
    check_whole_append(c, t, d, q_rot, D)
    assert d["T"].cpu().tolist() == [a + b for a, b in zip(T, new)]


@pytest.mark.parametrize("varlen", [False, True])
@pytest.mark.parametrize("rot", [0, 16, 64, 96])
def test_append_partial_rotation(av, varlen, rot):
    T = [3, 33, 64]
    new = [1, 1, 1] if not varlen else [20, 1, 33]
    c = H.make_cache(T, new, 2, 128, 32, True, seed=rot)
    t = new_tokens(c, 4, seed=rot + 1)
    d, q_rot, err = run_append(av, c, t, varlen, rot=rot, theta=500000.0)
    assert err == 0
    check_whole_append(c, t, d, q_rot, rot, 500000.0)


@pytest.mark.parametrize("varlen", [False, True])
def test_append_far_positions(av, varlen):
    """A page table of a million tokens; only the pages that get rows need to be named."""
    T, page = [999_983, 131_071], 16
    c = H.make_cache([0, 0], [1, 1], 2, 128, page, True, seed=11)
    c["T"] = torch.tensor(T, dtype=torch.int32)
    c["new"] = [17, 2] if varlen else [1, 1]
    num = 8
    for name in ("k", "v"):
        c[name] = torch.zeros(num, 2, page, 128).to(H.F8)
        c[name + "_scales"] = torch.full((num, 2), 112, dtype=torch.uint8)
    c["table"] = torch.full((2, 70_000), -1, dtype=torch.int32)
    for b in range(2):
        for i in range(3):
            c["table"][b, T[b] // page + i] = 3 * b + i
    t = new_tokens(c, 2, seed=12)
    d, q_rot, err = run_append(av, c, t, varlen)
    assert err == 0
    check_whole_append(c, t, d, q_rot, 128)


@pytest.mark.parametrize("varlen", [False, True])
def test_append_scale_grows_and_keeps(av, varlen):
    """Rows before a page's new ones take the larger scale; smaller new rows keep the present one."""
    page, D = 32, 128
    T = [31, 20, 7, 1]
    new = [1] * 4 if not varlen else [2, 5, 1, 31]
    for factor in (1e-3, 1.0, 40.0, 3e4):
        c = H.make_cache(T, new, 2, D, page, True, seed=21)
        t = new_tokens(c, 2, seed=22)
        t["k"] = (t["k"].float() * factor).clamp(-60000, 60000).half()
        t["v"] = (t["v"].float() * factor).clamp(-60000, 60000).half()
        d, q_rot, err = run_append(av, c, t, varlen)
        assert err == 0
        check_whole_append(c, t, d, q_rot, D)


@pytest.mark.parametrize("varlen", [False, True])
def test_append_zero_infinite_and_nan_rows(av, varlen):
    page, D = 16, 64
    T = [16, 16, 16, 3]
    new = [1] * 4 if not varlen else [3] * 4
    c = H.make_cache(T, new, 1, D, page, True, seed=31)
    t = new_tokens(c, 1, seed=32)
    first = [int(x) for x in t["cu"][:-1]]
    t["v"][first[0]: first[0] + new[0]] = 0.0
    t["v"][first[1], 0, 5] = float("inf")
    t["v"][first[2], 0, 6] = float("nan")
    t["v"][first[3], 0, 7] = float("-inf")
    d, q_rot, err = run_append(av, c, t, varlen)
    assert err == 0
    after = H.back(d)
    val = lambda b, at: P.values(after["v"], after["v_scales"], int(c["table"][b, at // page]), 0)[at % page]  # noqa: E731
    sc = lambda b: int(after["v_scales"][int(c["table"][b, int(T[b]) // page]), 0]) - 127  # noqa: E731
    assert sc(0) == -15 and (val(0, 16) == 0).all()
    assert sc(1) == 8 and float(val(1, 16)[5]) == 448.0 * 256
    assert math.isnan(float(val(2, 16)[6])) and not val(2, 16)[:6].isnan().any()
    assert sc(2) <= 0, "a NaN takes no part in the scale"
    assert sc(3) == 8 and float(val(3, 3)[7]) == -448.0 * 256


def test_append_out_of_room_and_bad_pages(av):
    """What does not fit, or has no page, is reported and not written; the other sequences are served."""
    page, D = 16, 128
    T, new = [10, 20, 5], [1, 1, 1]
    c = H.make_cache(T, new, 2, D, page, True, seed=41)
    c["table"] = c["table"][:, :2].contiguous()
    c["T"] = torch.tensor([10, 32, 5], dtype=torch.int32)  # sequence 1: both pages are full
    t = new_tokens(c, 2, seed=42)
    d, _, err = run_append(av, c, t, varlen=False, advance=True)
    assert err == CAPACITY and d["T"].cpu().tolist() == [11, 32, 6]
    after = H.back(d)
    assert torch.equal(H.bits(after["k"])[c["table"][1].long()], H.bits(c["k"])[c["table"][1].long()])
    for wrong in (-1, c["k"].shape[0], 2 ** 31 - 1, -2 ** 31):
        c = H.make_cache(T, new, 2, D, page, True, seed=43)
        c["table"][1, 1] = wrong
        t = new_tokens(c, 2, seed=44)
        for varlen in (False, True):
            d, _, err = run_append(av, c, t, varlen)
            assert err == PAGE_ERR
            changed = (H.bits(H.back(d)["k"]) != H.bits(c["k"])).any(3).any(2).any(1).nonzero().flatten().tolist()
            assert set(changed) == {int(c["table"][0, 0]), int(c["table"][2, 0])}


# ---------------------------------------------------------------- decode

def run_decode(av, c, t, append=True, advance=False, rot=-1, scale=None, ws=None, d=None):
    d = d or H.to_device(c)
    q = t["q"].to(DEV)
    B, hq, D = q.shape
    ws = ws if ws is not None else av.make_paged_workspace(B, hq, c["hkv"], D, B)
    out, q_rot = torch.full_like(q, float("nan")), torch.zeros_like(q)
    kw = dict(k_new=t["k"].to(DEV), v_new=t["v"].to(DEV)) if append else {}
    av.paged_decode(q, d["k"], d["v"], out, d["table"], d["T"], k_scales=d["k_scales"], v_scales=d["v_scales"],
                    scale=-1.0 if scale is None else scale, rotary_dim=rot, advance=advance, q_rot_out=q_rot, workspace=ws, **kw)
    torch.cuda.synchronize()
    return d, out.cpu(), q_rot.cpu(), av.paged_read_error(ws)


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("D,page,hkv,group,layout", [
    (128, 16, 2, 1, "hnd"), (128, 64, 2, 8, "nhd"), (128, 32, 1, 16, "hnd"), (64, 128, 2, 5, "sliced"),
    (64, 16, 1, 16, "hnd"), (256, 64, 1, 8, "hnd"), (256, 16, 2, 3, "nhd"), (128, 128, 1, 11, "sliced")])
def test_decode(av, e4m3, D, page, hkv, group, layout):
    T = [0, 1, 15, 16, 63, 64, 127, 128, 129, 300, 777]
    c = H.make_cache(T, [1] * len(T), hkv, D, page, e4m3, seed=D + page + group, layout=layout)
    t = new_tokens(c, hkv * group, seed=51)
    d, out, q_rot, err = run_decode(av, c, t, advance=True)
    assert err == 0
    check_whole_append(c, t, d, q_rot, D)
    after = H.back(d)
    H.check_attention(out, rotated_queries(t), after, c["table"], [x + 1 for x in T], range(len(T)), D ** -0.5, "decode")
    assert d["T"].cpu().tolist() == [x + 1 for x in T]


@pytest.mark.parametrize("e4m3", [True, False])
def test_decode_without_new_rows(av, e4m3):
    """Attention over what is cached; a sequence that holds nothing gives zeros."""
    T = [0, 1, 16, 17, 200]
    c = H.make_cache(T, [0] * len(T), 2, 128, 16, e4m3, seed=61)
    c["new"] = [1] * len(T)
    t = new_tokens(c, 6, seed=62)
    d, out, q_rot, err = run_decode(av, c, t, append=False)
    assert err == 0 and torch.equal(q_rot, t["q"])
    after = H.back(d)
    for name in "kv":
        assert torch.equal(H.bits(after[name]), H.bits(c[name]))
    assert (out[0] == 0).all()
    H.check_attention(out, t["q"].double(), c, c["table"], T, range(len(T)), 128 ** -0.5, "decode")


def test_decode_long_and_ragged(av):
    """Sequences cut over many CTAs beside ones of a single key."""
    T = [9000, 0, 1, 4097, 2, 2500]
    c = H.make_cache(T, [1] * len(T), 1, 128, 64, True, seed=71)
    t = new_tokens(c, 4, seed=72)
    d, out, q_rot, err = run_decode(av, c, t, scale=0.05)
    assert err == 0
    H.check_attention(out, rotated_queries(t), H.back(d), c["table"], [x + 1 for x in T], range(len(T)), 0.05, "decode")


def test_decode_sharp_scores_and_uneven_scales(av):
    """Scores far apart, and pages whose scales differ by 2^20: neither loses the small ones."""
    T = [200, 333]
    c = H.make_cache(T, [1, 1], 2, 128, 16, True, seed=81)
    g = torch.Generator().manual_seed(82)
    for name in "kv":
        e = torch.randint(-14, 7, c[name + "_scales"].shape, generator=g)
        c[name + "_scales"] = (e + 127).to(torch.uint8)
    t = new_tokens(c, 4, seed=83)
    d, out, q_rot, err = run_decode(av, c, t, scale=1e-6)
    H.check_attention(out, rotated_queries(t), H.back(d), c["table"], [x + 1 for x in T], [0, 1], 1e-6, "flat")
    c["k_scales"].fill_(127)
    d, out, q_rot, err = run_decode(av, c, t, scale=1.0)
    assert err == 0
    H.check_attention(out, rotated_queries(t), H.back(d), c["table"], [x + 1 for x in T], [0, 1], 1.0, "sharp")


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("gap", [8.0, 11.0, 14.0])
def test_decode_one_key_beside_many_small(av, e4m3, gap):
    """One key takes most of a row's attention and thousands share the rest: the small weights still count."""
    T = 12000
    c = H.make_cache([T], [0], 1, 128, 64, e4m3, seed=84)
    c["new"] = [1]
    t = new_tokens(c, 2, seed=85)
    u = torch.zeros(128)
    u[0] = 1.0
    for name in "kv":  # keys orthogonal to the query but for one; values of one sign, so that a lost mass shows
        raw = torch.zeros(c[name].shape) if name == "k" else torch.ones(c[name].shape) * 0.75
        if e4m3:
            c[name + "_scales"].fill_(127)
        if name == "k":
            page, row = int(c["table"][0, 31]), 17
            raw[page, 0, row] = u * 8.0
        else:
            page, row = int(c["table"][0, 31]), 17
            raw[page, 0, row] = -1.0
        c[name] = raw.to(c[name].dtype)
    t["q"] = (u * 8.0).half().expand(1, 2, 128).contiguous()
    d, out, q_rot, err = run_decode(av, c, t, append=False, scale=gap / 64.0)
    assert err == 0
    H.check_attention(out, t["q"].double(), c, c["table"], [T], [0], gap / 64.0, "sink")


def test_decode_bad_page_and_capacity(av):
    T = [50, 40, 30]
    for wrong in (-1, 10 ** 9):
        c = H.make_cache(T, [1] * 3, 2, 128, 16, True, seed=91)
        c["table"][1, 1] = wrong
        t = new_tokens(c, 4, seed=92)
        d, out, q_rot, err = run_decode(av, c, t)
        assert err == PAGE_ERR
        rows = [0, 2]
        H.check_attention(out[rows], rotated_queries(t)[rows], H.back(d), c["table"], [51, 31], rows, 128 ** -0.5, "others")
        assert not out[1].isnan().any()
    c = H.make_cache(T, [1] * 3, 2, 128, 16, True, seed=93)
    c["T"] = torch.tensor([50, 16 * c["table"].shape[1], -5], dtype=torch.int32)
    t = new_tokens(c, 4, seed=94)
    d, out, q_rot, err = run_decode(av, c, t, advance=True)
    assert err == CAPACITY and d["T"].cpu().tolist() == [51, 16 * c["table"].shape[1], -5]
    assert (out[1:] == 0).all()
    H.check_attention(out[:1], rotated_queries(t)[:1], H.back(d), c["table"], [51], [0], 128 ** -0.5, "the one that fits")


@pytest.mark.parametrize("e4m3,D", [(True, 128), (True, 64), (False, 128)])
def test_decode_many_short_sequences(av, e4m3, D):
    """More sequences than CTAs, most of a few keys and some long: units of every kind on one CTA."""
    T = [(7 * i) % 40 for i in range(331)] + [1500, 0, 700]
    c = H.make_cache(T, [1] * len(T), 1, D, 16, e4m3, seed=131)
    t = new_tokens(c, 2, seed=132)
    d, out, q_rot, err = run_decode(av, c, t, advance=True)
    assert err == 0 and d["T"].cpu().tolist() == [x + 1 for x in T]
    H.check_attention(out, rotated_queries(t), H.back(d), c["table"], [x + 1 for x in T], range(len(T)), D ** -0.5, "many")


@pytest.mark.parametrize("e4m3", [True, False])
def test_decode_largest_queries(av, e4m3):
    """Queries whose rotation passes fp16's range."""
    c = H.make_cache([33, 200], [1, 1], 1, 128, 32, e4m3, seed=133)
    t = new_tokens(c, 2, seed=134)
    t["q"] = (torch.sign(t["q"].float()) * 65504.0).half()
    d, out, q_rot, err = run_decode(av, c, t, scale=1e-6)
    assert err == 0 and rotated_queries(t).abs().max() > 70000
    H.check_attention(out, rotated_queries(t), H.back(d), c["table"], [34, 201], [0, 1], 1e-6, "largest")


@pytest.mark.parametrize("D,e4m3", [(128, True), (64, True), (128, False)])
@pytest.mark.parametrize("T", [[40, 40, 40], [3000, 40, 3000]])
def test_decode_nan_in_live_rows(av, D, e4m3, T):
    """A NaN among the keys that a row sees makes the row NaN, one among the values its dim, and neither anything else."""
    c = H.make_cache(T, [1] * 3, 2, D, 16, e4m3, seed=137)
    t = new_tokens(c, 4, seed=138)
    nan = torch.tensor(0x7F, dtype=torch.uint8).view(H.F8) if e4m3 else torch.tensor(float("nan"), dtype=torch.float16)
    raw = lambda x: x.view(torch.uint8) if e4m3 else x  # noqa: E731
    raw(c["k"])[int(c["table"][0, 1]), 1, 3, 7] = raw(nan)   # sequence 0, kv head 1, row 19
    raw(c["v"])[int(c["table"][2, 2]), 0, 5, 9] = raw(nan)   # sequence 2, kv head 0, row 37, dim 9
    d, out, q_rot, err = run_decode(av, c, t)
    assert err == 0
    want = torch.zeros(out.shape, dtype=torch.bool)
    want[0, 2:] = True
    want[2, :2, 9] = True
    assert torch.equal(out.isnan(), want)


@pytest.mark.parametrize("D,e4m3", [(128, True), (64, True), (128, False)])
def test_decode_queries_that_are_not_finite(av, D, e4m3):
    c = H.make_cache([200, 300], [1] * 2, 2, D, 16, e4m3, seed=139)
    t = new_tokens(c, 4, seed=140)
    t["q"][0, 1, 5] = float("inf")
    t["q"][1, 2, 6] = float("nan")
    d, out, q_rot, err = run_decode(av, c, t)
    assert err == 0
    want = torch.zeros(out.shape, dtype=torch.bool)
    want[0, 1] = want[1, 2] = True
    assert torch.equal(out.isnan(), want)


@pytest.mark.parametrize("D,e4m3", [(128, True), (64, True), (128, False)])
def test_decode_refused_sequence_keeps_q_rot(av, D, e4m3):
    c = H.make_cache([50, 40, 30], [1] * 3, 2, D, 16, e4m3, seed=141)
    c["T"] = torch.tensor([50, 16 * c["table"].shape[1], -5], dtype=torch.int32)
    d, out, q_rot, err = run_decode(av, c, new_tokens(c, 4, seed=142))
    assert err == CAPACITY and (q_rot[0] != 0).any() and (q_rot[1:] == 0).all() and (out[1:] == 0).all()


@pytest.mark.parametrize("theta", [0.3, 1.0, 5e5, 1e30])
def test_append_odd_thetas(av, theta):
    c = H.make_cache([1000, 3], [1, 1], 1, 64, 16, False, seed=135)
    t = new_tokens(c, 1, seed=136)
    d, q_rot, err = run_append(av, c, t, varlen=False, theta=theta)
    assert err == 0
    # the entry points take theta in fp32
    check_whole_append(c, t, d, q_rot, 64, float(torch.tensor(theta, dtype=torch.float32)))


def test_decode_shared_prefix_pages(av):
    """Two sequences that name the same full pages read the same rows."""
    c = H.make_cache([64, 64], [1, 1], 2, 128, 16, True, seed=101)
    c["table"][1, :4] = c["table"][0, :4]
    t = new_tokens(c, 4, seed=102)
    d, out, q_rot, err = run_decode(av, c, t)
    assert err == 0
    H.check_attention(out, rotated_queries(t), H.back(d), c["table"], [65, 65], [0, 1], 128 ** -0.5, "shared")


# ---------------------------------------------------------------- prefill

def run_prefill(av, c, t, advance=False, rot=-1, ws=None, max_new=None):
    d = H.to_device(c)
    q, k, v = t["q"].to(DEV), t["k"].to(DEV), t["v"].to(DEV)
    out = torch.full_like(q, 7.0)
    B, hq, D = len(c["new"]), q.shape[1], q.shape[2]
    most = max_new or max(c["new"])
    if ws is None:
        ws = av.make_paged_workspace(B, hq, c["hkv"], D, q.shape[0], most, sum(c["new"]) + int(c["T"].clamp(min=0).sum()))
    av.paged_prefill(q, k, v, d["k"], d["v"], out, d["table"], d["T"], t["cu"].to(DEV), most, k_scales=d["k_scales"],
                     v_scales=d["v_scales"], rotary_dim=rot, advance=advance, workspace=ws)
    torch.cuda.synchronize()
    return d, out.cpu(), av.paged_read_error(ws)


def check_prefill(c, t, d, out, rot=128):
    """The pools as an append leaves them, and causal attention over them (long chunks hold the queries in fp16)."""
    n = len(t["pos"])
    after = H.back(d)
    H.check_append(c, after, "k", c["T"], t["cu"], c["table"], exact_rotation(t["k"][:n], t["pos"], rot), rot > 0)
    H.check_append(c, after, "v", c["T"], t["cu"], c["table"], t["v"][:n].double(), False)
    seq = [b for b, m in enumerate(c["new"]) for _ in range(m)]
    q = rotated_queries(t, rot)
    H.check_attention(out[:n], q, after, c["table"], [p + 1 for p in t["pos"]], seq, 128 ** -0.5, "prefill", q_fp16=True)
    assert (out[n:] == 7.0).all(), "rows behind the last sequence were written"


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("page,hkv,group,T,new,layout", [
    (16, 2, 1, [0, 30, 17], [5, 1, 0], "hnd"),
    (64, 1, 8, [100, 0, 63], [3, 1, 2], "nhd"),
    (32, 2, 4, [0, 200], [130, 40], "hnd"),
    (128, 1, 2, [1, 127, 0, 129], [128, 129, 300, 1], "sliced"),
    (16, 1, 16, [0, 77, 0], [19, 0, 260], "hnd"),
    (64, 1, 3, [500], [257], "nhd")])
def test_prefill(av, e4m3, page, hkv, group, T, new, layout):
    c = H.make_cache(T, new, hkv, 128, page, e4m3, seed=page + group, layout=layout)
    t = new_tokens(c, hkv * group, seed=111, gap=4)
    d, out, err = run_prefill(av, c, t, advance=True)
    assert err == 0
    check_prefill(c, t, d, out)
    assert d["T"].cpu().tolist() == [a + b for a, b in zip(T, new)]


def test_prefill_out_of_room(av):
    """A sequence that does not fit, a bound on n_b that is broken, a page that is none: reported, others served."""
    c = H.make_cache([0, 10, 0], [40, 300, 20], 1, 128, 16, True, seed=121)
    t = new_tokens(c, 2, seed=122)
    d, out, err = run_prefill(av, c, t, advance=True, max_new=40)
    assert err == CAPACITY and d["T"].cpu().tolist() == [40, 10, 20]
    seq = [0] * 40 + [2] * 20
    rows = list(range(40)) + list(range(340, 360))
    pos = list(range(40)) + list(range(20))
    q = exact_rotation(t["q"][rows], pos, 128)
    H.check_attention(out[rows], q, H.back(d), c["table"], [p + 1 for p in pos], seq, 128 ** -0.5, "others", q_fp16=True)
    assert (out[40:340] == 7.0).all()
    for new in ([40, 3], [100, 90]):
        c = H.make_cache([40, 17], new, 1, 128, 16, True, seed=123)
        c["table"][1, 1] = c["k"].shape[0]
        t = new_tokens(c, 2, seed=124)
        d, out, err = run_prefill(av, c, t)
        assert err == PAGE_ERR
        q = rotated_queries(t)[: new[0]]
        H.check_attention(out[: new[0]], q, H.back(d), c["table"], [p + 1 for p in t["pos"][: new[0]]], [0] * new[0],
                          128 ** -0.5, "others", q_fp16=True)
