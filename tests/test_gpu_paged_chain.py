"""Chains of paged steps without an ordinary launch between them, as a captured loop over layers makes them."""
import pytest
import torch

from helpers import randn_half

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    import fully_custom_cuda_inference_lamma2_b200 as pkg

    return pkg


@pytest.mark.parametrize("dtype,D", [(torch.float8_e4m3fn, 128), (torch.float8_e4m3fn, 64), (torch.float16, 128)])
@pytest.mark.parametrize("with_append", [False, True])
def test_early_reads_right_behind_a_step_that_advances(pkg, dtype, D, with_append):
    """Step after step of several layers: the last layer's call moves the lengths, the next step's first call waits for it,
    and the calls behind that one read lengths and rows early. Eager and captured, the same bits as without early reads."""
    L, B, hq, hkv, steps = 4, 3, 4, 2, 40
    T = [0, 250, 1003]
    got = []
    for early, use_graph in ((False, False), (True, False), (True, True)):
        cache = pkg.PagedKVCache(L, B, hkv, D, num_pages=120, page_size=16, q_heads=hq, dtype=dtype)
        for t in (cache.k, cache.v):
            t.view(torch.uint8 if dtype != torch.float16 else torch.int16).fill_(0x3A if dtype != torch.float16 else 0x3800)
        if cache.k_scales is not None:
            cache.k_scales.view(torch.uint8).fill_(124)
            cache.v_scales.view(torch.uint8).fill_(124)
        for b in range(B):
            cache.reserve(b, T[b] + steps + 2)
        cache.seq_lens.copy_(torch.tensor(T, dtype=torch.int32))
        q, k, v = (randn_half((L, B, h, D), 501 + i).cuda() for i, h in enumerate((hq, hkv, hkv)))
        out = torch.zeros(steps, L, B, hq, D, dtype=torch.float16, device="cuda")

        def chain():
            for i in range(steps):
                for l in range(L):
                    if with_append and l == L - 1:  # the step's last call is an append that moves the lengths
                        pkg.paged_decode(cache, l, q[l], out[i, l], prefetch_kv=early)
                        pkg.paged_append(cache, l, k[l], v[l], advance=True)
                    else:
                        pkg.paged_decode(cache, l, q[l], out[i, l], k_new=k[l], v_new=v[l], advance=(l == L - 1),
                                         prefetch_kv=early and l > 0)

        if use_graph:
            graph = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(graph, stream=side):
                chain()
            graph.replay()
        else:
            chain()
        torch.cuda.synchronize()
        assert cache.read_error() == 0 and cache.seq_lens.tolist() == [t + steps for t in T]
        got.append((out.clone(), cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone()))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)
