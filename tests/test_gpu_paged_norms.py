"""GPU results of the paged attention calls as a whole, in the 2-norm against 64 bits: a part of a query or of a weight that
went missing shows here (tests/paged_norms.py has the bounds)."""
import pytest
import torch

import paged_helpers as H
import paged_norms as N
from test_gpu_paged import new_tokens, rotated_queries, run_decode
from test_gpu_paged_edges import prefill, seq_of_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def av():
    import fully_custom_cuda_inference_lamma2_b200 as pkg

    return pkg.attn_varlen


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("D,page,group", [(128, 16, 1), (128, 64, 8), (128, 32, 16), (64, 128, 4), (64, 16, 16), (256, 32, 8)])
@pytest.mark.parametrize("wide", [False, True])
def test_decode(av, e4m3, D, page, group, wide):
    T = [300, 777, 64, 4000, 1500]
    scale = N.WIDE if wide else D ** -0.5
    c = N.plain_cache(T, 2, D, page, e4m3, seed=611)
    t = new_tokens(c, 2 * group, seed=612)
    d, out, q_rot, err = run_decode(av, c, t, scale=scale)
    assert err == 0
    want = N.exact(rotated_queries(t), H.back(d), c["table"], [n + 1 for n in T], range(len(T)), scale)
    assert N.off(out, want) < N.SPLIT


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("group,new", [(1, [5, 1, 64]), (4, [3, 16, 2]), (8, [8, 1, 5]), (16, [4, 1, 3])])
@pytest.mark.parametrize("wide", [False, True])
def test_short_chunks(av, e4m3, group, new, wide):
    T = [900, 2000, 40]
    scale = N.WIDE if wide else 128 ** -0.5
    c = N.plain_cache(T, 2, 128, 32, e4m3, seed=613, spare_rows=max(new))
    c["new"] = new
    t = new_tokens(c, 2 * group, seed=614)
    d, out, err = prefill(av, c, t, scale=scale)
    assert err == 0 and max(new) * group <= 64
    want = N.exact(rotated_queries(t), H.back(d), c["table"], [p + 1 for p in t["pos"]], seq_of_rows(c), scale)
    assert N.off(out, want) < N.SPLIT


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("hkv,group,T,new", [
    (1, 4, [0, 900, 37], [300, 20, 129]),
    (2, 8, [6000, 0, 129, 3000, 1], [700, 1, 2300, 512, 0]),   # rings of many tiles, several items a sequence and head
    (8, 1, [130 * i % 1700 for i in range(40)], [(91 * i) % 400 + 1 for i in range(40)]),  # more items than CTAs
])
def test_long_chunks(av, e4m3, hkv, group, T, new):
    c = N.plain_cache(T, hkv, 128, 64, e4m3, seed=615, spare_rows=max(new))
    c["new"] = new
    t = new_tokens(c, hkv * group, seed=616)
    d, out, err = prefill(av, c, t, advance=True)
    assert err == 0 and max(new) * group > 64 and d["T"].cpu().tolist() == [a + b for a, b in zip(T, new)]
    # every row of short calls, else some of each sequence: its first and last, and those around ends of tiles and items
    n = len(t["pos"])
    seq = seq_of_rows(c)
    rows = range(n)
    if n > 600:
        g = torch.Generator().manual_seed(617)
        starts = [sum(new[:b]) for b in range(len(new))]
        edges = [s + i for s, m in zip(starts, new) for i in (0, 1, 127, 128, 255, 256, 257, m - 1) if 0 <= i < m]
        rows = sorted(set(edges) | set(torch.randint(0, n, (150,), generator=g).tolist()))
    rows = list(rows)
    want = N.exact(rotated_queries(t)[rows], H.back(d), c["table"], [t["pos"][r] + 1 for r in rows], [seq[r] for r in rows], 128 ** -0.5)
    assert N.off(out[rows], want) < N.LONG
    assert not (out[:n] == 7.0).all(-1).any()
    # ... and row by row, so that none hides behind the others
    worst = ((out[rows].double() - want).norm(dim=-1) / want.norm(dim=-1)).max()
    assert worst < 4 * N.LONG, float(worst)
