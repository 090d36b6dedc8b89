"""The paged operators as they are used: together, captured, in streams, through PagedKVCache and the greedy decoder."""
import pytest
import torch

import paged_helpers as H
from helpers import randn_half
from oracle import llama_oracle as LO
from oracle import paged_oracle as P
from test_gpu_paged import exact_rotation

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    import fully_custom_cuda_inference_lamma2_b200 as pkg

    return pkg


def snapshot(cache, layer):
    k, v, ks, vs = cache.layer(layer)
    return H.back(dict(k=k, v=v, k_scales=ks, v_scales=vs))


def rows(shape, seed):
    return randn_half(shape, seed).cuda()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float16])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (4, 4)])
def test_prompts_then_steps_then_a_proposal(pkg, dtype, hq, hkv):
    """Ragged prompts (two layers), captured decode steps over page ends, a chunk of a few proposed tokens, and one
    sequence that leaves while another takes its pages."""
    D, page, B = 128, 16, 3
    lens = [70, 5, 33]
    cache = pkg.PagedKVCache(2, B, hkv, D, num_pages=24, page_size=page, q_heads=hq, dtype=dtype, max_tokens=160, max_seqlen=80)
    for b, n in enumerate(lens):
        cache.reserve(b, n + 20)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
    n = sum(lens)
    q, k, v = rows((2, n, hq, D), 1), rows((2, n, hkv, D), 2), rows((2, n, hkv, D), 3)
    out = torch.empty_like(q)
    for l in range(2):
        pkg.paged_prefill(cache, l, q[l], k[l], v[l], out[l], cu, max(lens), advance=(l == 1))
    torch.cuda.synchronize()
    assert cache.seq_lens.tolist() == lens and cache.read_error() == 0
    table = cache.page_table.cpu()
    pos = [i for m in lens for i in range(m)]
    seq = [b for b, m in enumerate(lens) for _ in range(m)]
    for l in range(2):
        H.check_attention(out[l].cpu(), exact_rotation(q[l].cpu(), pos, D), snapshot(cache, l), table, [p + 1 for p in pos],
                          seq, D ** -0.5, f"prompt, layer {l}", q_fp16=True)

    # one graph for every step: its inputs are refilled, the lengths move on the device
    qs, ks, vs = rows((2, B, hq, D), 4), rows((2, B, hkv, D), 5), rows((2, B, hkv, D), 6)
    o = torch.zeros_like(qs)

    def step():
        for l in range(2):
            pkg.paged_decode(cache, l, qs[l], o[l], k_new=ks[l], v_new=vs[l], advance=(l == 1))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    before = cache.seq_lens.clone()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    cache.seq_lens.copy_(before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(page + 2):
        for j, t in enumerate((qs, ks, vs)):
            t.copy_(rows(t.shape, 100 + 3 * i + j) * (1.0 + 0.3 * i))
        graph.replay()
        torch.cuda.synchronize()
        now = [m + i for m in lens]
        assert cache.seq_lens.tolist() == [m + 1 for m in now]
        if i % 5 == 0 or i == page + 1:
            for l in range(2):
                exact = torch.stack([P.rope(qs[l, b].cpu(), now[b], D, 10000.0) for b in range(B)])
                H.check_attention(o[l].cpu(), exact, snapshot(cache, l), table, [m + 1 for m in now], range(B), D ** -0.5,
                                  f"step {i}, layer {l}")
    assert cache.read_error() == 0

    # sequence 1 leaves; its pages serve sequence 0, and the freed table row is never followed
    held = set(cache.pages_of(1))
    cache.release(1)
    cache.reserve(0, lens[0] + 20 + page)
    assert set(cache.pages_of(0)) & held
    new = [2, 0, 1]
    at = [lens[0] + page + 2, 0, lens[2] + page + 2]
    m = sum(new)
    cu = torch.tensor([0, 2, 2, 3], dtype=torch.int32).cuda()
    q, k, v = rows((m, hq, D), 7), rows((m, hkv, D), 8), rows((m, hkv, D), 9)
    out = torch.empty_like(q)
    pkg.paged_prefill(cache, 0, q, k, v, out, cu, 2)
    torch.cuda.synchronize()
    pos, seq = [at[0], at[0] + 1, at[2]], [0, 0, 2]
    H.check_attention(out.cpu(), exact_rotation(q.cpu(), pos, D), snapshot(cache, 0), cache.page_table.cpu(),
                      [p + 1 for p in pos], seq, D ** -0.5, "proposal")
    assert cache.seq_lens.tolist() == [at[0], 0, at[2]] and cache.read_error() == 0


def test_cache_bookkeeping(pkg):
    cache = pkg.PagedKVCache(1, 2, 1, 64, num_pages=5, page_size=16, max_pages=4, dtype=torch.float16)
    cache.reserve(0, 17)
    cache.reserve(1, 33)
    assert len(cache.pages_of(0)) == 2 and len(cache.pages_of(1)) == 3 and cache.free_pages() == 0
    cache.reserve(0, 32)  # has them
    with pytest.raises(RuntimeError, match="free"):
        cache.reserve(0, 33)
    assert len(cache.pages_of(0)) == 2
    cache.release(1)
    assert cache.free_pages() == 3 and (cache.page_table[1] == -1).all()
    cache.reserve(0, 64)
    with pytest.raises(RuntimeError, match="pages"):
        cache.reserve(0, 65)
    got = cache.page_table[0].tolist()
    assert got == cache.pages_of(0) and len(set(got)) == 4


def test_calls_in_two_streams_with_their_own_workspaces(pkg):
    """Two caches stepped at once on two streams, and a call on another stream than the tensors were made on."""
    av = pkg.attn_varlen
    cases = []
    for i in range(2):
        c = H.make_cache([900 + 37 * i, 40, 2000], [1] * 3, 2, 128, 32, bool(i), seed=201 + i)
        t = dict(q=rows((3, 6, 128), 210 + i), k=rows((3, 2, 128), 220 + i), v=rows((3, 2, 128), 230 + i))
        cases.append((c, t, H.to_device(c), av.make_paged_workspace(3, 6, 2, 128, 3), torch.cuda.Stream(), torch.zeros(3, 6, 128).half().cuda()))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, t, d, ws, s, out in cases:
            with torch.cuda.stream(s):
                av.paged_decode(t["q"], d["k"], d["v"], out, d["table"], d["T"], k_scales=d["k_scales"],
                                v_scales=d["v_scales"], k_new=t["k"], v_new=t["v"], workspace=ws)
    torch.cuda.synchronize()
    for c, t, d, ws, s, out in cases:
        T = c["T"].tolist()
        exact = torch.stack([P.rope(t["q"][b].cpu(), T[b], 128, 10000.0) for b in range(3)])
        H.check_attention(out.cpu(), exact, H.back(d), c["table"], [x + 1 for x in T], range(3), 128 ** -0.5, "stream")
        assert av.paged_read_error(ws) == 0


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float16])
def test_early_reads_change_nothing(pkg, dtype):
    """A chain of layers' steps with and without prefetch_kv, over a page end, eager and replayed: the same bits."""
    L, B, hq, hkv, D, steps = 6, 5, 8, 2, 128, 20
    T = [0, 13, 500, 1300, 31]
    got = []
    for early, use_graph in ((False, False), (True, False), (True, True)):
        cache = pkg.PagedKVCache(L, B, hkv, D, num_pages=140, page_size=16, q_heads=hq, dtype=dtype)
        for t in (cache.k, cache.v):
            t.view(torch.uint8 if dtype != torch.float16 else torch.int16).fill_(0x3A if dtype != torch.float16 else 0x3800)
        if cache.k_scales is not None:
            cache.k_scales.view(torch.uint8).fill_(124)
            cache.v_scales.view(torch.uint8).fill_(124)
        for b in range(B):
            cache.reserve(b, T[b] + steps + 2)
        cache.seq_lens.copy_(torch.tensor(T, dtype=torch.int32))
        q, k, v = rows((L, B, hq, D), 301), rows((L, B, hkv, D), 302), rows((L, B, hkv, D), 303)
        out = torch.zeros(L, B, hq, D).half().cuda()

        def step():
            q.mul_(1.01)  # an ordinary launch between the steps
            for l in range(L):
                pkg.paged_decode(cache, l, q[l], out[l], k_new=k[l], v_new=v[l], advance=(l == L - 1), prefetch_kv=early)

        seen = []
        if use_graph:
            step()
            seen.append(out.clone())
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
        for _ in range(steps - len(seen)):
            graph.replay() if use_graph else step()
            seen.append(out.clone())
        torch.cuda.synchronize()
        assert cache.read_error() == 0 and cache.seq_lens.tolist() == [t + steps for t in T]
        got.append((torch.stack(seen), cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone()))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)


def test_one_workspace_serves_calls_of_other_shapes(pkg):
    """Append, decode, prompts and short chunks of different batches through one workspace, in turn, twice."""
    av = pkg.attn_varlen
    ws = av.make_paged_workspace(4, 16, 2, 128, 400, 200, 2000)
    for _ in range(2):
        for T, new, hq in (([5, 0, 100], [1, 1, 1], 4), ([5, 0], [150, 40], 4), ([1000], [1], 16), ([30, 64, 2, 9], [2, 1, 3, 1], 4)):
            c = H.make_cache(T, new, 2, 128, 16, True, seed=240)
            n = sum(new)
            q, k, v = rows((n, hq, 128), 241), rows((n, 2, 128), 242), rows((n, 2, 128), 243)
            d, out = H.to_device(c), torch.zeros(n, hq, 128).half().cuda()
            cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32).cuda()
            if max(new) == 1:
                av.paged_decode(q, d["k"], d["v"], out, d["table"], d["T"], k_scales=d["k_scales"], v_scales=d["v_scales"],
                                k_new=k, v_new=v, workspace=ws)
            else:
                av.paged_prefill(q, k, v, d["k"], d["v"], out, d["table"], d["T"], cu, max(new), k_scales=d["k_scales"],
                                 v_scales=d["v_scales"], workspace=ws)
            pos = [T[b] + i for b, m in enumerate(new) for i in range(m)]
            seq = [b for b, m in enumerate(new) for _ in range(m)]
            H.check_attention(out.cpu(), exact_rotation(q.cpu(), pos, 128), H.back(d), c["table"], [p + 1 for p in pos], seq,
                              128 ** -0.5, "shared workspace", q_fp16=True)
            assert av.paged_read_error(ws) == 0


@pytest.mark.parametrize("rot", [0, 32, 96])
def test_partial_rotation_of_every_call(pkg, rot):
    av = pkg.attn_varlen
    for T, new in (([40, 3, 0], [1, 1, 1]), ([40, 3, 0], [3, 1, 2]), ([40, 3, 0], [70, 1, 90])):
        c = H.make_cache(T, new, 1, 128, 32, True, seed=310)
        n = sum(new)
        q, k, v = rows((n, 4, 128), 311), rows((n, 1, 128), 312), rows((n, 1, 128), 313)
        d, out = H.to_device(c), torch.zeros(n, 4, 128).half().cuda()
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32).cuda()
        kw = dict(k_scales=d["k_scales"], v_scales=d["v_scales"], rotary_dim=rot, rope_theta=1000.0)
        if max(new) == 1:
            av.paged_decode(q, d["k"], d["v"], out, d["table"], d["T"], k_new=k, v_new=v, **kw)
        else:
            av.paged_prefill(q, k, v, d["k"], d["v"], out, d["table"], d["T"], cu, max(new), **kw)
        pos = [T[b] + i for b, m in enumerate(new) for i in range(m)]
        seq = [b for b, m in enumerate(new) for _ in range(m)]
        after = H.back(d)
        H.check_append(c, after, "k", c["T"], cu.cpu(), c["table"], exact_rotation(k.cpu(), pos, rot, 1000.0), rot > 0)
        H.check_attention(out.cpu(), exact_rotation(q.cpu(), pos, rot, 1000.0), after, c["table"], [p + 1 for p in pos], seq,
                          128 ** -0.5, f"rot {rot}", q_fp16=max(new) > 16)


@pytest.mark.parametrize("e4m3", [True, False])
def test_strided_operands_and_a_full_cache(pkg, e4m3):
    """q, k and v as slices of one projection, a page table and scales that are slices too, T + 1 = capacity, and
    no workspace given, under capture: its own is zeroed at every replay."""
    av = pkg.attn_varlen
    B, hq, hkv, D, page = 3, 6, 2, 64, 16
    T = [3 * page - 1, 2 * page, 7]
    c = H.make_cache(T, [1] * B, hkv, D, page, e4m3, seed=320)
    d = H.to_device(c)
    wide = torch.full((B, 9), -1, dtype=torch.int32).cuda()
    wide[:, 2:5] = d["table"][:, :3]
    table = wide[:, 2:5]
    if e4m3:
        for name in ("k_scales", "v_scales"):
            s = d[name].view(torch.uint8)
            both = torch.full((s.shape[1], 2, s.shape[0]), 200, dtype=torch.uint8).cuda()
            both[:, 1] = s.t()
            d[name] = both[:, 1].t().view(torch.float8_e8m0fnu)
    qkv = rows((B, (hq + 2 * hkv) * D), 321).view(B, hq + 2 * hkv, D)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    o2 = torch.zeros(B, hq, 2, D).half().cuda()
    out = o2[:, :, 1]
    kw = dict(k_scales=d["k_scales"], v_scales=d["v_scales"], k_new=k, v_new=v)
    av.paged_decode(q, d["k"], d["v"], out, table, d["T"], **kw)
    first = out.clone()
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        av.paged_decode(q, d["k"], d["v"], out, table, d["T"], **kw)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first) and (o2[:, :, 0] == 0).all()
    exact = torch.stack([P.rope(q[b].cpu(), T[b], D, 10000.0) for b in range(B)])
    after = H.back({n: (t if not (e4m3 and n.endswith("scales")) else t.view(torch.uint8).contiguous().view(torch.float8_e8m0fnu))
                    for n, t in d.items()})
    H.check_attention(out.cpu(), exact, after, c["table"], [t + 1 for t in T], range(B), D ** -0.5, "slices")


@pytest.mark.parametrize("page,D,e4m3", [(64, 128, True), (16, 64, False)])
def test_offsets_past_32_bits(pkg, page, D, e4m3):
    """Pages behind 4 GB of a pool, read, appended to, expanded."""
    av = pkg.attn_varlen
    T, new = [130, 5], [1, 1]
    c = H.make_cache(T, new if D != 128 else [80, 3], 2, D, page, e4m3, seed=330)
    small = H.to_device(c)
    num = c["k"].shape[0]
    total = (5 << 30) // (2 * page * D * (1 if e4m3 else 2))
    d = dict(small)
    for name in ("k", "v"):
        big = torch.empty((total,) + tuple(c[name].shape[1:]), dtype=torch.uint8 if e4m3 else torch.float16, device="cuda")
        big[-num:] = small[name].view(big.dtype)
        d[name] = big.view(small[name].dtype)
        if e4m3:
            sc = torch.full((total, 2), 127, dtype=torch.uint8, device="cuda")
            sc[-num:] = small[name + "_scales"].view(torch.uint8)
            d[name + "_scales"] = sc.view(torch.float8_e8m0fnu)
    table = torch.where(small["table"] >= 0, small["table"] + (total - num), small["table"])

    def tail():
        return H.back({n: (t[-num:] if n != "table" and n != "T" and t is not None else t) for n, t in d.items()})

    kw = dict(k_scales=d["k_scales"], v_scales=d["v_scales"])
    q, k, v = rows((2, 4, D), 331), rows((2, 2, D), 332), rows((2, 2, D), 333)
    out = torch.zeros_like(q)
    av.paged_decode(q, d["k"], d["v"], out, table, d["T"], k_new=k, v_new=v, **kw)
    exact = torch.stack([P.rope(q[b].cpu(), T[b], D, 10000.0) for b in range(2)])
    H.check_attention(out.cpu(), exact, tail(), c["table"], [t + 1 for t in T], range(2), D ** -0.5, "far decode")
    if D == 128:
        cu = torch.tensor([0, 80, 83], dtype=torch.int32).cuda()
        q, k, v = rows((83, 4, D), 334), rows((83, 2, D), 335), rows((83, 2, D), 336)
        out = torch.zeros_like(q)
        av.paged_prefill(q, k, v, d["k"], d["v"], out, table, d["T"], cu, 80, max_kv_tokens=300, **kw)
        pos = [T[0] + i for i in range(80)] + [T[1] + i for i in range(3)]
        H.check_attention(out.cpu(), exact_rotation(q.cpu(), pos, D), tail(), c["table"], [p + 1 for p in pos], [0] * 80 + [1] * 3,
                          D ** -0.5, "far prefill", q_fp16=True)


def test_thousands_of_sequences_and_too_many(pkg):
    """A batch whose bookkeeping takes a good part of shared memory, and one that it does not hold: refused."""
    av = pkg.attn_varlen
    for B, fits in ((3000, True), (20000, False)):
        pool = torch.full((8, 1, 16, 128), 0x30, dtype=torch.uint8).cuda().view(torch.float8_e4m3fn)
        vals = torch.full((8, 1, 16, 128), 0x38, dtype=torch.uint8).cuda().view(torch.float8_e4m3fn)  # 1.0
        scales = torch.full((8, 1), 127, dtype=torch.uint8).cuda().view(torch.float8_e8m0fnu)
        table = (torch.arange(B * 2, dtype=torch.int32) % 8).view(B, 2).cuda()  # pages shared by many: read only
        lens = (torch.arange(B, dtype=torch.int32) % 33).cuda()
        q, out = rows((B, 2, 128), 340), torch.full((B, 2, 128), 7.0).half().cuda()
        call = lambda: av.paged_decode(q, pool, vals, out, table, lens, k_scales=scales, v_scales=scales)  # noqa: E731
        if not fits:
            with pytest.raises(RuntimeError, match="batch too large"):
                call()
            continue
        call()
        torch.cuda.synchronize()
        want = (lens > 0).half()[:, None, None].expand_as(out)  # values are all 1: the mean is 1, or 0 of none
        assert torch.equal(out, want)


def test_prefill_of_rows_that_belong_to_nobody(pkg):
    """Offsets that name no row of the batch, and ones that run backwards: nothing is written, the latter is reported."""
    av = pkg.attn_varlen
    c = H.make_cache([20, 0], [90, 0], 1, 128, 16, True, seed=350)
    d = H.to_device(c)
    q, k = rows((100, 2, 128), 351), rows((100, 1, 128), 352)
    ws = av.make_paged_workspace(2, 2, 1, 128, 100, 90, 400)
    for offsets, err in (([0, 0, 0], 0), ([0, -3, 2], 1), ([0, 200, 200], 1), ([60, 60, 10], 1)):
        out = torch.full_like(q, 7.0)
        av.paged_prefill(q, k, k, d["k"], d["v"], out, d["table"], d["T"], torch.tensor(offsets, dtype=torch.int32).cuda(), 90,
                         k_scales=d["k_scales"], v_scales=d["v_scales"], workspace=ws)
        torch.cuda.synchronize()
        assert av.paged_read_error(ws) == err, offsets
        assert (out == 7.0).all() and torch.equal(H.bits(H.back(d)["k"]), H.bits(c["k"]))


def test_entry_points_refuse_what_does_not_fit(pkg):
    av = pkg.attn_varlen
    c = H.make_cache([5, 6], [1, 1], 2, 128, 16, True, seed=250)
    d = H.to_device(c)
    q, k = rows((2, 4, 128), 251), rows((2, 2, 128), 252)
    out = torch.empty_like(q)
    good = dict(k_scales=d["k_scales"], v_scales=d["v_scales"], k_new=k, v_new=k)
    call = lambda q=q, out=out, kp=d["k"], table=d["table"], lens=d["T"], **kw: av.paged_decode(  # noqa: E731
        q, kp, d["v"], out, table, lens, **{**good, **kw})
    call()
    with pytest.raises(RuntimeError, match="k_scales"):
        call(k_scales=None)
    with pytest.raises(RuntimeError, match="k_scales"):
        call(k_scales=d["k_scales"][:-1])
    with pytest.raises(RuntimeError, match="go together"):
        call(v_new=None)
    with pytest.raises(RuntimeError, match="advance"):
        call(k_new=None, v_new=None, advance=True)
    with pytest.raises(RuntimeError, match="one type"):
        call(kp=torch.zeros(d["k"].shape).half().cuda())
    with pytest.raises(RuntimeError, match="fp16"):
        call(q=q.float())
    with pytest.raises(RuntimeError, match="out must be"):
        call(out=out[:, :2])
    with pytest.raises(RuntimeError, match="int32"):
        call(table=d["table"].long())
    with pytest.raises(RuntimeError, match="one entry per page_table row"):
        call(lens=d["T"][:1])
    with pytest.raises(RuntimeError, match="one new token per sequence"):
        call(q=q[:1], out=out[:1])
    with pytest.raises(RuntimeError, match="16-byte"):
        call(q=torch.zeros(2 * 4 * 128 + 1).half().cuda()[1:].view(2, 4, 128))
    with pytest.raises(RuntimeError, match="workspace"):
        call(workspace=torch.zeros(4096, dtype=torch.uint8).cuda())
    with pytest.raises(RuntimeError, match="no scales"):
        h = torch.zeros(d["k"].shape).half().cuda()
        av.paged_decode(q, h, h, out, d["table"], d["T"], **good)
    with pytest.raises(RuntimeError, match="max_seqlen_q"):
        av.paged_append(k, k, d["k"], d["v"], d["table"], d["T"], k_scales=d["k_scales"], v_scales=d["v_scales"],
                        cu_seqlens_q=torch.tensor([0, 1, 2], dtype=torch.int32).cuda())
    with pytest.raises(RuntimeError, match="room"):
        n = 80
        av.paged_prefill(rows((n, 4, 128), 1), rows((n, 2, 128), 2), rows((n, 2, 128), 3), d["k"], d["v"],
                         torch.empty(n, 4, 128).half().cuda(), d["table"], d["T"], torch.tensor([0, 40, 80], dtype=torch.int32).cuda(), 40,
                         k_scales=d["k_scales"], v_scales=d["v_scales"], max_kv_tokens=0)


def test_empty_calls(pkg):
    """No new tokens: nothing is launched, nothing is written."""
    av = pkg.attn_varlen
    c = H.make_cache([5, 0], [0, 0], 2, 128, 16, True, seed=260)
    d = H.to_device(c)
    z = lambda h: torch.empty(0, h, 128).half().cuda()  # noqa: E731
    cu = torch.zeros(3, dtype=torch.int32).cuda()
    before = av.launch_count()
    av.paged_prefill(z(4), z(2), z(2), d["k"], d["v"], z(4), d["table"], d["T"], cu, 0, k_scales=d["k_scales"], v_scales=d["v_scales"])
    av.paged_append(z(2), z(2), d["k"], d["v"], d["table"], d["T"], k_scales=d["k_scales"], v_scales=d["v_scales"],
                    cu_seqlens_q=cu, max_seqlen_q=0, q=z(4), q_rot_out=z(4))
    torch.cuda.synchronize()
    assert av.launch_count() == before and torch.equal(H.bits(H.back(d)["k"]), H.bits(c["k"]))


@pytest.mark.parametrize("kv_cache", ["paged", "paged_e4m3"])
def test_greedy_decoder_on_pages(pkg, kv_cache):
    """The decoder on pages: fp16 pages within the fp32 oracle's bound for an fp16 model (relative L2 2e-2); for both
    kinds graph replays equal eager steps bit for bit, also over page ends and for a prompt that fills the cache again."""
    from fully_custom_cuda_inference_lamma2_b200.llama_decode import GreedyDecoder, LlamaShape, LlamaWeights

    shape = LlamaShape(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, intermediate=1024, vocab=1000)
    w = LlamaWeights(shape, seed=3, std=0.05)
    prompt = torch.randint(0, shape.vocab, (45,), generator=torch.Generator().manual_seed(4))
    seen = []
    for use_graph in (True, False):
        dec = GreedyDecoder(w, capacity=96, max_new_tokens=64, kv_cache=kv_cache, page_size=16)
        for _ in range(2):
            dec.arena.seq_lens.zero_()
            dec.prefill(prompt.cuda())
            logits, toks = [dec.logits.float().cpu().clone()], [int(dec.token.item())]
            if use_graph and dec.graph is None:
                dec.capture()
            for _ in range(20):
                dec.graph.replay() if use_graph else dec._step()
                logits.append(dec.logits.float().cpu().clone())
                toks.append(int(dec.token.item()))
            assert int(dec.arena.seq_lens.item()) == 65 and dec.arena.read_error() == 0
            seen.append((torch.stack(logits), toks))
    for logits, toks in seen[1:]:
        assert toks == seen[0][1] and torch.equal(logits, seen[0][0])
    if kv_cache == "paged":
        ref = LO.logits_for(w, prompt.tolist() + seen[0][1][:-1])[prompt.numel() - 1:]
        assert float((seen[0][0] - ref).norm() / ref.norm()) < 2e-2
    with pytest.raises(ValueError):
        GreedyDecoder(w, capacity=8, kv_cache="pages")
