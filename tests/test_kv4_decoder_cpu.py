"""Gemma4SyntheticDecoder.step refuses what does not fit the cache before the cache's state moves on: a
refused step can be put right and made again. The plan is a stand-in (there is no CPU path)."""
import pytest
import torch

from gemma_triton_flash_attn import gemma4_synthetic as g4
from gemma_triton_flash_attn.kv4 import KV4Plan


def config(**kw):
    args = dict(vocab_size=64, hidden_size=64, num_layers=3, global_every=3, global_heads=2, global_kv_heads=1,
                global_head_dim=128, local_heads=2, local_kv_heads=2, local_head_dim=64, sliding_window=8,
                intermediate_size=64)
    return g4.Gemma4SyntheticConfig(**(args | kw))


def cache_for(cfg, batch=2, **kw):
    return g4.DecoderKV4Cache(cfg, batch, 128, page_size=16, device="cpu", **kw)


@pytest.mark.parametrize("what,error,match", [
    ("batch", ValueError, "rows"), ("empty", ValueError, "token"), ("shape", ValueError, "2-D"),
    ("new_lens", ValueError, "new_lens"), ("dtype", TypeError, "dtype"), ("layers", ValueError, "layers"),
    ("heads", ValueError, "layer 0")])
def test_a_refused_step_leaves_the_cache_as_it_was(what, error, match, monkeypatch):
    planned = []

    def plan(kv_lens, new_lens, block_table, free_pages, free_state, page_size, max_new):
        planned.append(new_lens)
        return KV4Plan(block_table + 1, kv_lens + 1, new_lens, torch.zeros(2, max_new, dtype=torch.int32),
                       torch.zeros(2, max_new, dtype=torch.int32), free_state + 1, torch.ones(2))

    monkeypatch.setattr(g4, "kv4_plan", plan)
    cfg = config()
    model = g4.Gemma4SyntheticDecoder(cfg).to(torch.bfloat16)
    cache, ids, new = cache_for(cfg), torch.zeros(2, 3, dtype=torch.long), torch.ones(2, dtype=torch.int32)
    if what == "batch":
        ids = ids[:1]
    if what == "empty":
        ids = ids[:, :0]
    if what == "shape":
        ids = ids[0]
    if what == "new_lens":
        new = new[:1]
    if what == "dtype":
        cache = cache_for(cfg, dtype=torch.float16)
    if what == "layers":
        cache = cache_for(config(num_layers=2))
    if what == "heads":
        cache = cache_for(config(local_kv_heads=1))
    kept = [t.clone() for t in (cache.block_table, cache.kv_lens, cache.free_state, cache.free_pages)]
    with pytest.raises(error, match=match):
        model.step(ids, new, cache)
    assert not planned
    for t, k in zip((cache.block_table, cache.kv_lens, cache.free_state, cache.free_pages), kept):
        assert torch.equal(t, k)


def test_a_cache_for_no_tokens_is_refused():
    for kw in (dict(max_batch=0, max_len=16), dict(max_batch=1, max_len=0), dict(max_batch=1, max_len=16, page_size=24)):
        with pytest.raises((ValueError, NotImplementedError)):
            g4.DecoderKV4Cache(config(), device="cpu", **kw)
