"""The greedy decoder on pages: what capturing its step leaves behind."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def snapshot(cache, rows):
    """What the cache holds of the first `rows` rows of its sequence, and its pages' scales, bit for bit."""
    if not hasattr(cache, "pages_of"):
        return [cache.layer(l)[i][0, :, :rows].clone() for l in range(2) for i in range(2)]
    pages = cache.pages_of(0)[: -(-rows // cache.page_size)]
    got = []
    for pool, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        raw = pool.view(torch.uint8)[:, pages].transpose(2, 3)  # [L, pages, page, Hkv, bytes]
        got.append(raw.flatten(1, 2)[:, :rows].clone())
        if scales is not None:
            got.append(scales.view(torch.uint8)[:, pages].clone())
    return got


@pytest.mark.parametrize("kv_cache", ["arena", "paged", "paged_e4m3"])
@pytest.mark.parametrize("warmup", [0, 12])
@pytest.mark.parametrize("other", [False, True])
def test_capture_leaves_the_cache_as_it_was(kv_cache, warmup, other):
    """Steps run to warm up before the capture are taken back, the pages that they wrote too: a captured decoder goes on as
    one that steps eagerly, also when the next token is another one than capture saw."""
    from fully_custom_cuda_inference_lamma2_b200.llama_decode import GreedyDecoder, LlamaShape, LlamaWeights

    shape = LlamaShape(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, intermediate=1024, vocab=1000)
    w = LlamaWeights(shape, seed=3, std=0.05)
    # a token whose value in layer 0, kv head 0, is far above the others'
    w.embed[17] = w.w_qkv[0, (shape.heads + shape.kv_heads) * shape.head_dim]
    prompt = torch.randint(100, shape.vocab, (37,), generator=torch.Generator().manual_seed(4))
    seen = []
    for captured in (False, True):
        dec = GreedyDecoder(w, capacity=96, max_new_tokens=64, kv_cache=kv_cache, page_size=16)
        dec.prefill(prompt.cuda())
        first = dec.token.clone()
        if captured:
            if other:
                dec.token.fill_(17)
            at = (dec.arena.seq_lens.clone(), dec.token.clone(), dec.step_idx.clone())
            held = snapshot(dec.arena, 37)
            dec.capture(warmup=warmup)
            assert all(torch.equal(a, b) for a, b in zip(held, snapshot(dec.arena, 37)))
            assert all(torch.equal(a, b) for a, b in zip(at, (dec.arena.seq_lens, dec.token, dec.step_idx)))
            dec.token.copy_(first)
        logits, toks = [], []
        for _ in range(20):
            dec.graph.replay() if captured else dec._step()
            logits.append(dec.logits.clone())
            toks.append(int(dec.token.item()))
        assert dec.arena.seq_lens.tolist() == [57]
        seen.append((torch.stack(logits), toks, dec.generated[:20].tolist()))
    assert seen[0][1:] == seen[1][1:] and torch.equal(seen[0][0], seen[1][0])
