"""The paged 4-bit KV cache on the GPU against 64-bit references (kv4_ref.py): plan, append, read and
attention, each alone and as a serving loop runs them, with the bounds derived there."""
import math

import numpy as np
import pytest
import torch

import gemma_triton_flash_attn as gfa
import kv4_ref
from gemma_triton_flash_attn import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "").replace(" ", "")  # noqa: E731


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    assert _lib.device_status(torch.cuda.current_device(), reset=True) == 0, "a kernel recorded a status"


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(DEV)


def rand(shape, seed, dtype, factor=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * factor).to(dtype)


# ------------------------------------------------------------------ plan
def _plan_inputs(B, cols, page, max_new, seed, spare, kinds):
    r = np.random.RandomState(seed)
    lens = r.randint(0, cols * page + 1, B)
    lens[r.rand(B) < 0.2] = 0
    new = np.where(r.rand(B) < 0.5, 1, r.randint(0, max_new + 3, B))  # some beyond max_new
    if kinds == "mixed":
        new[r.rand(B) < 0.3] = -1
    used = -(-lens // page)
    total = int(used.sum()) + spare
    perm = r.permutation(total + 5)
    table = np.full((B, cols), -1)
    at = 0
    for b in range(B):
        table[b, :used[b]] = perm[at:at + used[b]]
        at += used[b]
    F = total + 5
    head = r.randint(F)
    free = np.full(F, -1)
    free[(head + np.arange(spare)) % F] = perm[at:at + spare]
    return lens, new, table, free, np.array([head, spare])


@pytest.mark.parametrize("B,cols,page,max_new,spare", [
    (1, 1, 16, 1, 1), (1, 3, 64, 200, 0), (8, 64, 64, 1, 8), (33, 5, 16, 40, 20), (257, 7, 32, 100, 64),
    (600, 3, 256, 3, 1), (64, 33, 128, 777, 10000)])
@pytest.mark.parametrize("kinds", ["grow", "mixed"])
def test_plan_matches_the_loop(B, cols, page, max_new, spare, kinds):
    for seed in range(3):
        lens, new, table, free, state = _plan_inputs(B, cols, page, max_new, seed, spare, kinds)
        want = kv4_ref.plan(lens, new, table, free, state, page, max_new)
        wide = i32(np.concatenate([table, np.full((B, 2), 7)], 1))[:, :cols]  # rows with a stride of their own
        args = [i32(lens), i32(new), wide, i32(free), i32(state)]
        kept = [a.clone() for a in args]
        got = gfa.kv4_plan(*args, page_size=page, max_new=max_new)
        for name in got._fields:
            assert np.array_equal(getattr(got, name).cpu().numpy(), want[name]), name
        assert np.array_equal(args[3].cpu().numpy(), want["free_pages"])
        for a, b in zip(args[:3] + args[4:], kept[:3] + kept[4:]):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ append and read
def scattered_table(B, cols, total, seed):
    return i32(np.random.RandomState(seed).permutation(total)[:B * cols].reshape(B, cols))


def slots_of(table, start, n, new, page):
    pos = np.asarray(start)[:, None] + np.arange(n)[None]
    t = table.cpu().numpy()
    s = np.take_along_axis(t, np.minimum(pos // page, t.shape[1] - 1), 1) * page + pos % page
    return i32(np.where(np.arange(n)[None] < np.asarray(new)[:, None], s, -1))


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("B,H,N,page", [(1, 1, 1, 16), (2, 3, 37, 16), (3, 2, 70, 64), (1, 4, 300, 256)])
def test_append_writes_the_format_and_read_returns_it(D, dtype, B, H, N, page):
    start = [5 + 13 * b for b in range(B)]
    new = [N - b for b in range(B)] if N > 3 else [N] * B
    cols = -(-(max(start) + N) // page)
    total = B * cols + 2
    cache = gfa.kv4_alloc(total, H, D, page, dtype, DEV)
    cache.pages.fill_(0xFF)
    table = scattered_table(B, cols, total, 3)
    slots = slots_of(table, start, N, new, page)
    k = rand((B, N, H, D), 1, dtype).to(DEV).transpose(1, 2)  # strided, as a projection leaves it
    v = rand((B, N, H, D), 2, dtype, 30.0).to(DEV).transpose(1, 2)
    before = cache.pages.clone()
    gfa.kv4_append(cache, k, v, slots)
    want = [kv4_ref.values(*kv4_ref.quantise(x.cpu())) for x in (k, v)]
    held = kv4_ref.unpack(cache.pages, H, D, page)
    untouched = kv4_ref.unpack(before, H, D, page)
    sl = slots.cpu().numpy()
    for b in range(B):
        for i in range(N):
            if sl[b, i] < 0:
                continue
            for kind in range(2):
                assert np.array_equal(held[sl[b, i], kind], want[kind][b, :, i].numpy()), (b, i, kind)
    others = np.setdiff1d(np.arange(total * page), sl[sl >= 0])
    assert np.array_equal(held[others], untouched[others], equal_nan=True)  # the other slots are as they were
    lens = i32(np.asarray(start) + np.asarray(new))
    for n in (N, N + 9):
        rk, rv = gfa.kv4_read(cache, table, lens, n, starts=i32(start))
        for got, w in zip((rk, rv), want):
            assert got.shape == (B, H, n, D) and got.dtype == dtype
            for b in range(B):
                assert torch.equal(got[b, :, :new[b]].cpu().double(), w[b, :, :new[b]])
                assert (got[b, :, new[b]:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_quantised_values_at_the_borders_of_the_type(dtype):
    """Zeros, constants, one-sided and tiny groups, the largest numbers, ties: exactly the definition."""
    most, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [torch.zeros(64), torch.full((64,), 3.0), torch.full((64,), -0.75), torch.arange(64.) * 0.25,
            torch.linspace(-7.5, 7.5, 64), torch.linspace(-most, most, 64), torch.linspace(0, most, 64),
            torch.linspace(-tiny, tiny, 64), torch.full((64,), tiny / 8), torch.linspace(100, 101, 64),
            torch.arange(64.) % 16 * 0.5 - 3.75, torch.full((64,), most), torch.full((64,), -most)]
    x = torch.stack(rows).to(dtype)
    x = torch.cat([x, rand((243, 64), 9, dtype, 1.0) * torch.exp2(torch.arange(243.) % 30 - 15)[:, None].to(dtype)])
    # (linspace from -most overflows its own step in fp32 at bf16's largest: that group holds infinities)
    x = torch.cat([x, torch.linspace(-1, 1, 16 * 64).reshape(16, 64).flip(0).to(dtype) * most,
                   torch.linspace(-1, 1, 64).to(dtype).expand(16, 64) * most])
    x = x.reshape(1, 1, -1, 64)
    n = x.shape[2]
    cache = gfa.kv4_alloc(n // 16, 1, 64, 16, dtype, DEV)
    table = i32(np.arange(n // 16))[None]
    slots = i32(np.arange(n))[None]
    gfa.kv4_append(cache, x.to(DEV), x.flip(2).to(DEV), slots)
    k, v = gfa.kv4_read(cache, table, i32([n]), n)
    want = kv4_ref.values(*kv4_ref.quantise(x))
    fine = torch.isfinite(x).all(-1, keepdim=True)
    assert torch.equal(torch.isfinite(want), fine.expand_as(want))
    assert np.array_equal(k.cpu().double().numpy(), want.numpy(), equal_nan=True)
    assert np.array_equal(v.cpu().double().numpy(), want.flip(2).numpy(), equal_nan=True)
    # half a step from the value, a whole one where the zero point's rounding cuts the last code
    # (or the type's largest number does)
    c, s, z = kv4_ref.quantise(x)
    err = (want - x.double()).abs().unflatten(-1, (-1, 64)).amax(-1)
    assert (err <= s)[fine].all()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_groups_that_are_not_finite_read_back_as_nan(dtype):
    x = rand((1, 2, 16, 128), 4, dtype)
    x[0, 0, 3, 5], x[0, 1, 7, 64], x[0, 1, 8, 127] = math.inf, -math.inf, math.nan
    cache = gfa.kv4_alloc(1, 2, 128, 16, dtype, DEV)
    gfa.kv4_append(cache, x.to(DEV), x.to(DEV), i32(np.arange(16))[None])
    want = kv4_ref.values(*kv4_ref.quantise(x))
    for got in gfa.kv4_read(cache, i32([[0]]), i32([16]), 16):
        assert np.array_equal(got.cpu().double().numpy(), want.numpy(), equal_nan=True)
    assert int(torch.isnan(want).sum()) == 3 * 64


# ------------------------------------------------------------------ attention
def filled(B, H, D, L, page, dtype, seed, factor=1.0):
    """A cache with L random tokens for each of B requests, its table, and the values held (float64)."""
    cols = -(-L // page)
    total = B * cols + 1
    cache = gfa.kv4_alloc(total, H, D, page, dtype, DEV)
    cache.pages.random_(0, 256, generator=torch.Generator(DEV).manual_seed(seed))  # stale slots hold anything
    table = scattered_table(B, cols, total, seed)
    k, v = (rand((B, H, L, D), seed + i, dtype, factor).to(DEV) for i in range(2))
    gfa.kv4_append(cache, k, v, slots_of(table, [0] * B, L, [L] * B, page))
    held = [kv4_ref.values(*kv4_ref.quantise(x)) for x in (k, v)]
    return cache, table, held


def check(q, cache, table, held, lens, q_lens, causal, window, scale=None):
    B, Hq, N, D = q.shape
    full = q_lens is None
    o, lse = gfa.attention_flash_gqa_kv4(q, cache, table, i32(lens), causal=causal, slide_size=window,
                                         q_lens=None if full else i32(q_lens), softmax_scale=scale, return_lse=True)
    plain = gfa.attention_flash_gqa_kv4(q, cache, table, i32(lens), causal=causal, slide_size=window,
                                        q_lens=None if full else i32(q_lens), softmax_scale=scale)
    assert torch.equal(o, plain)
    assert o.dtype == q.dtype and o.shape == q.shape
    ql = [N] * B if full else q_lens
    want, wl, bound = kv4_ref.attention(q, *held, lens, ql, causal, window, D ** -0.5 if scale is None else scale)
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all()
    assert (err <= bound).all(), f"error {err.max():.3e}, over the bound by {(err - bound).max():.3e}"
    seen = ~torch.isinf(wl)
    assert torch.equal(torch.isinf(lse), ~seen)
    if seen.any():
        assert (lse.double() - wl)[seen].abs().max() <= 1e-4 * (1 + wl[seen].abs().max())
    return o, lse


SHAPES = [
    # B, Hq, Hkv, N, lens, q_lens, page, causal, window
    (1, 1, 1, 1, [1], None, 16, True, 0),
    (2, 8, 1, 1, [17, 1], None, 16, True, 0),
    (3, 16, 8, 1, [1000, 511, 513], None, 64, True, 512),
    (4, 8, 2, 1, [0, 700, 128, 129], None, 32, True, 0),            # an empty request
    (2, 14, 2, 1, [2000, 77], None, 128, True, 0),                  # 7 query heads a group
    (3, 8, 4, 5, [5, 300, 640], [5, 3, 0], 64, True, 0),            # verification, ragged, no rows
    (2, 4, 2, 9, [1030, 9], [9, 9], 256, True, 100),
    (2, 8, 8, 3, [515, 40], None, 16, False, 0),                    # every row sees all keys
    (2, 6, 2, 33, [400, 33], [33, 20], 64, True, 0),                # several row tiles
    (1, 8, 1, 20, [10], [10], 64, True, 3),
    (1, 4, 4, 7, [900], None, 64, True, 1),                         # each row sees only itself
    (2, 4, 1, 4, [2, 50], [4, 4], 16, True, 0),                     # more rows than keys: the first see nothing
]


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "B{}_H{}-{}_N{}_L{}_q{}_p{}_c{}_w{}".format(*s).replace(" ", ""))
def test_attention_within_the_rounding_bound(D, dtype, shape):
    B, Hq, Hkv, N, lens, q_lens, page, causal, window = shape
    cache, table, held = filled(B, Hkv, D, max(max(lens), 1), page, dtype, 11)
    q = rand((B, N, Hq, D), 5, dtype).to(DEV).transpose(1, 2)
    o, lse = check(q, cache, table, held, lens, q_lens, causal, window)
    for b in range(B):
        n = N if q_lens is None else q_lens[b]
        assert (o[b, :, n:] == 0).all() and torch.isinf(lse[b, :, n:]).all()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("N,capacity", [(3, 704), (3, 65536), (40, 704)])  # short tiles, and long ones twice
@pytest.mark.parametrize("window", [0, 300])
def test_tiles_of_few_and_of_many_blocks(D, dtype, N, capacity, window):
    """The length of a tile goes by the table's capacity and the rows: partial tiles at either end of both."""
    B, Hkv, page = 5, 4, 16
    cache, table, held = filled(B, Hkv, D, 700, page, dtype, 21)
    wide = torch.full((B, capacity // page), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = rand((B, 8, N, D), 7, dtype).to(DEV)
    check(q, cache, wide, held, [700, 513, 1, 128, 0], [N, 1, N, 2, N], True, window)


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.float16),
                                     (512, torch.bfloat16)], ids=ids)
def test_attention_over_a_long_ragged_batch(D, dtype):
    lens = [9000, 1, 4097, 0, 12345]
    cache, table, held = filled(5, 2, D, 12345, 64, dtype, 21)
    q = rand((5, 8, 2, D), 6, dtype, 2.0).to(DEV)
    check(q, cache, table, held, lens, [2, 1, 0, 2, 2], True, 0)
    check(q, cache, table, held, lens, None, True, 3000, scale=0.01)


# ------------------------------------------------------------------ many rows
CHUNKS = [
    # B, Hq, Hkv, N, lens, q_lens, page, causal, window
    (1, 4, 1, 130, [130], None, 64, True, 0),                        # a prompt with nothing before it
    (3, 8, 2, 200, [1000, 200, 300], [200, 77, 0], 16, True, 0),     # ragged, one request without rows
    (2, 4, 4, 150, [0, 150], [150, 150], 32, True, 0),               # nothing cached: zeros
    (2, 8, 4, 257, [2000, 600], [257, 129], 64, True, 300),          # window shorter than the cache
    (2, 4, 2, 128, [1500, 700], None, 128, True, 1),                 # each row sees only itself
    (2, 6, 2, 140, [600, 90], [140, 90], 64, False, 0),              # every row sees all keys
    (2, 4, 1, 150, [100, 700], [150, 150], 64, True, 0),             # more rows than keys
]


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", CHUNKS, ids=lambda s: "B{}_H{}-{}_N{}_L{}_q{}_p{}_c{}_w{}".format(*s).replace(" ", ""))
def test_chunks_within_the_rounding_bound(D, dtype, shape):
    B, Hq, Hkv, N, lens, q_lens, page, causal, window = shape
    cache, table, held = filled(B, Hkv, D, max(max(lens), 1), page, dtype, 31)
    q = rand((B, N, Hq, D), 7, dtype).to(DEV).transpose(1, 2)
    o, lse = check(q, cache, table, held, lens, q_lens, causal, window)
    for b in range(B):
        n = N if q_lens is None else q_lens[b]
        assert (o[b, :, n:] == 0).all() and torch.isinf(lse[b, :, n:]).all()


# enough rows for the dense path (keys and values written out, tcgen05 forward) at every head_dim
DENSE = [
    (3, 32, 4, 150, [1000, 150, 301], [150, 77, 0], 16, True, 0),
    (3, 32, 4, 160, [700, 160, 0], None, 64, True, 200),             # window, an empty request
    (2, 64, 4, 140, [90, 600], [140, 130], 32, False, 0),
    (4, 32, 4, 131, [256, 257, 131, 60], None, 128, True, 0),        # more rows than keys in the last one
]


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", DENSE, ids=lambda s: "B{}_H{}-{}_N{}_L{}_q{}_p{}_c{}_w{}".format(*s).replace(" ", ""))
def test_wide_chunks_within_the_rounding_bound(D, dtype, shape):
    test_chunks_within_the_rounding_bound(D, dtype, shape)


@pytest.mark.parametrize("window", [0, 300])
def test_chunks_of_more_requests_than_are_written_out_at_once(window):
    """Keys and values of two requests of 131072 tokens' room fill 2 GiB: five requests take three turns."""
    B, Hkv, D, page, N, capacity, dtype = 5, 4, 512, 256, 240, 131072, torch.bfloat16
    cache, table, held = filled(B, Hkv, D, 600, page, dtype, 31)
    wide = torch.full((B, capacity // page), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = rand((B, 32, N, D), 8, dtype).to(DEV)
    check(q, cache, wide, held, [600, 240, 513, 0, 257], [N, N, 7, 3, 130], True, window)
