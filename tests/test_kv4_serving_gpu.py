"""The paged 4-bit cache's operators together, as a serving loop runs them: a small Gemma-4-shaped decoder
steps through prompts, single tokens, drafted tokens and finished requests. Every attention call of
every layer is checked against a 64-bit computation over the keys and values that were appended for its
request so far; a captured step is replayed against eager ones."""
import pytest
import torch

import kv4_ref
from gemma_triton_flash_attn import _lib, gemma4_synthetic as g4

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert _lib.device_status(torch.cuda.current_device(), reset=True) == 0, "a kernel recorded a status"


def small_config():
    return g4.Gemma4SyntheticConfig(vocab_size=512, hidden_size=256, num_layers=3, global_every=3, global_heads=8,
                                    global_kv_heads=1, global_head_dim=128, local_heads=4, local_kv_heads=2,
                                    local_head_dim=64, sliding_window=40, intermediate_size=512)


def decoder(seed=0):
    cfg = small_config()
    return cfg, g4.Gemma4SyntheticDecoder(cfg).to(DEV).to(torch.bfloat16).init_weights(seed, 0.08)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# new tokens of four rows: prompts long and short, decoding, drafts, a row that finishes
# and one that takes its place, a request that the pool has no pages for
SCHEDULE = [
    ((150, 7, 0, 33), 150),
    ((1, 1, 0, 1), 1),
    ((1, 3, 60, 0), 60),
    ((4, 2, 1, 4), 4),
    ((1, -1, 1, 1), 1),
    ((1, 140, 1, 1), 140),
    ((1, 1, 1, 300), 300),  # refused
    ((2, 1, 0, 1), 2),
]


def test_serving_loop_matches_the_appended_history(monkeypatch):
    cfg, model = decoder()
    cache = g4.DecoderKV4Cache(cfg, 4, 640, num_pages=32, page_size=16)
    layer_of = {id(c): i for i, c in enumerate(cache.layers)}
    history = [[[None, None] for _ in range(4)] for _ in cache.layers]  # layer, row: values (H, t, D) float64
    lens = [0] * 4
    seen = []

    real_append, real_attend = g4.kv4_append, g4.attention_flash_gqa_kv4

    def append(c, k, v, slot_map):
        real_append(c, k, v, slot_map)
        for row in range(4):
            n = int((slot_map[row] >= 0).sum())
            for kind, x in enumerate((k, v)):
                held = kv4_ref.values(*kv4_ref.quantise(x[row, :, :n]))
                old = history[layer_of[id(c)]][row][kind]
                history[layer_of[id(c)]][row][kind] = held if old is None else torch.cat([old, held], 1)

    def attend(q, c, table, kv_lens, **kw):
        o = real_attend(q, c, table, kv_lens, **kw)
        rows = history[layer_of[id(c)]]
        L = max([1] + [r[0].shape[1] for r in rows if r[0] is not None])
        k, v = (torch.zeros(4, c.num_kv_heads, L, c.head_dim, dtype=torch.float64, device=DEV) for _ in range(2))
        for b, r in enumerate(rows):
            if r[0] is not None:
                k[b, :, :r[0].shape[1]], v[b, :, :r[1].shape[1]] = r[0], r[1]
        want, _, bound = kv4_ref.attention(q, k, v, kv_lens.tolist(), kw["q_lens"].tolist(), kw["causal"],
                                           kw["slide_size"], kw["softmax_scale"])
        assert ((o.double() - want).abs() <= bound).all()
        assert kv_lens.tolist() == [0 if r[0] is None else r[0].shape[1] for r in rows]
        seen.append(layer_of[id(c)])
        return o

    monkeypatch.setattr(g4, "kv4_append", append)
    monkeypatch.setattr(g4, "attention_flash_gqa_kv4", attend)
    g = torch.Generator().manual_seed(1)
    for step, (new, n) in enumerate(SCHEDULE):
        for row, add in enumerate(new):
            if add < 0:
                lens[row] = 0
                for h in history:
                    h[row] = [None, None]
        logits, plan = model.step(torch.randint(0, 512, (4, n), generator=g).to(DEV), ints(*new), cache)
        accepted = plan.accepted.tolist()
        assert accepted == [0 if (step == 6 and row == 3) else 1 for row in range(4)]
        for row, add in enumerate(new):
            if accepted[row] and add > 0:
                assert plan.positions[row, :add].tolist() == list(range(lens[row], lens[row] + add))
                lens[row] += add
        assert cache.kv_lens.tolist() == lens
        assert torch.isfinite(logits).all()
    assert seen == list(range(len(cache.layers))) * len(SCHEDULE)
    used = sum(-(-n // 16) for n in lens)
    assert int(cache.free_state[1]) == 32 - used
    held = cache.block_table[cache.block_table >= 0].tolist()
    ring = torch.roll(cache.free_pages, -int(cache.free_state[0]))[:32 - used].tolist()
    assert sorted(held + ring) == list(range(32))  # every page once


def test_captured_step_replays_as_eager_steps():
    cfg, model = decoder(3)
    caches = [g4.DecoderKV4Cache(cfg, 3, 512, page_size=32) for _ in range(2)]
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, 512, (3, 90), generator=g).to(DEV)
    for c in caches:
        model.step(prompt, ints(90, 17, 1), c)
    ids, new = torch.zeros(3, 1, dtype=torch.long, device=DEV), ints(1, 1, 1)
    # warm up on a third cache, then capture a step of caches[1]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        warm = g4.DecoderKV4Cache(cfg, 3, 512, page_size=32)
        for _ in range(2):
            model.step(ids, new, warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, _ = model.step(ids, new, caches[1])
    for step in range(70):  # over page borders, and past the window of the sliding layers
        ids.copy_(torch.randint(0, 512, (3, 1), generator=g).to(DEV))
        if step == 40:
            new.copy_(ints(1, 0, 1))
        eager, _ = model.step(ids, new, caches[0])
        graph.replay()
        assert torch.equal(eager, captured), step
        assert torch.equal(caches[0].kv_lens, caches[1].kv_lens)
    assert torch.equal(caches[0].block_table, caches[1].block_table)
    assert caches[0].kv_lens.tolist() == [160, 57, 71]
