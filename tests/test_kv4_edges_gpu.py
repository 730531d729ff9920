"""Edges of the paged 4-bit cache's operators: refusals that need CUDA tensors, entries that are out of
range, streams and graphs, shared and stale pages, non-finite values in masked places, the bounded waits."""
import math

import numpy as np
import pytest
import torch

import gemma_triton_flash_attn as gfa
import kv4_ref
from gemma_triton_flash_attn import _lib
from test_kv4_gpu import DEV, check, filled, i32, ids, rand, scattered_table, slots_of

pytestmark = pytest.mark.gpu
PAGE, SLOT, LENGTH = 16, 17, 18  # status codes, csrc/kv4_layout.cuh


def status():
    return _lib.device_status(torch.cuda.current_device(), reset=True)


@pytest.fixture(autouse=True)
def _status_clean():
    status()
    yield
    assert status() == 0, "a kernel recorded a status"


def small(dtype=torch.bfloat16, D=128, H=2, L=100, page=16, B=2, seed=3):
    cache, table, held = filled(B, H, D, L, page, dtype, seed)
    return cache, table, held


# ------------------------------------------------------------------ refusals
def test_refusals_of_cuda_tensors():
    cache, table, _ = small()
    lens, q = i32([100, 50]), rand((2, 4, 1, 128), 1, torch.bfloat16).to(DEV)
    att = gfa.attention_flash_gqa_kv4
    with pytest.raises(TypeError, match="dtype"):
        att(q.half(), cache, table, lens)
    with pytest.raises(TypeError, match="int32"):
        att(q, cache, table, lens.long())
    with pytest.raises(TypeError, match="int32"):
        att(q, cache, table.long(), lens)
    with pytest.raises(ValueError, match="block_table"):
        att(q, cache, table[:1], lens)
    with pytest.raises(ValueError, match="kv_lens"):
        att(q, cache, table, lens[:1])
    with pytest.raises(ValueError, match="q_lens"):
        att(q, cache, table, lens, q_lens=lens[:1])
    with pytest.raises(ValueError, match="4-D"):
        att(q[0], cache, table, lens)
    with pytest.raises(ValueError, match="head_dim"):
        att(q[..., :64], cache, table, lens)
    with pytest.raises(ValueError, match="multiple"):
        att(q[:, :3], cache, table, lens)
    with pytest.raises(ValueError, match="empty"):
        att(q[:, :, :0], cache, table, lens)
    with pytest.raises(ValueError, match="slide_size"):
        att(q, cache, table, lens, causal=True, slide_size=-2)
    with pytest.raises(ValueError, match="softmax_scale"):
        att(q, cache, table, lens, softmax_scale=-1.0)
    with pytest.raises(ValueError, match="max_kv_len"):
        att(q, cache, table, lens, max_kv_len=0)
    with pytest.raises(NotImplementedError, match="backward"):
        att(q.requires_grad_(), cache, table, lens)
    k = rand((2, 2, 3, 128), 2, torch.bfloat16).to(DEV)
    with pytest.raises(ValueError, match="shape"):
        gfa.kv4_append(cache, k, k[:, :, :2], i32(np.zeros((2, 3))))
    with pytest.raises(ValueError, match="shape"):
        gfa.kv4_append(cache, k[:, :1], k[:, :1], i32(np.zeros((2, 3))))
    with pytest.raises(ValueError, match="slot_map"):
        gfa.kv4_append(cache, k, k, i32(np.zeros((2, 4))))
    with pytest.raises(TypeError, match="dtype"):
        gfa.kv4_append(cache, k.half(), k.half(), i32(np.zeros((2, 3))))
    with pytest.raises(ValueError, match="rows"):
        gfa.kv4_read(cache, table, lens, 0)
    with pytest.raises(ValueError, match="starts"):
        gfa.kv4_read(cache, table, lens, 4, starts=lens[:1])
    z = i32([0, 0])
    with pytest.raises(ValueError, match="free_pages"):
        gfa.kv4_plan(z, z, table, i32(np.zeros((4, 2)))[:, 0], z, page_size=16, max_new=1)
    with pytest.raises(ValueError, match="max_new"):
        gfa.kv4_plan(z, z, table, i32(np.zeros(4)), z, page_size=16, max_new=0)
    with pytest.raises(NotImplementedError, match="page_size"):
        gfa.kv4_plan(z, z, table, i32(np.zeros(4)), z, page_size=20, max_new=1)


# ------------------------------------------------------------------ entries out of range
def test_slots_outside_the_cache_are_skipped_and_recorded():
    cache = gfa.kv4_alloc(2, 1, 64, 16, torch.float16, DEV)
    cache.pages.zero_()
    k = rand((1, 1, 5, 64), 1, torch.float16).to(DEV)
    gfa.kv4_append(cache, k, k, i32([[-1, 3, 32, 2 ** 31 - 1, -7]]))
    assert status() == SLOT
    got, _ = gfa.kv4_read(cache, i32([[0, 1]]), i32([32]), 32)
    want = kv4_ref.values(*kv4_ref.quantise(k))[0, 0, 1]
    assert torch.equal(got[0, 0, 3].double(), want)
    assert (got[0, 0, :3] == 0).all() and (got[0, 0, 4:] == 0).all()


@pytest.mark.parametrize("Hq,N", [(4, 1), (32, 150)])  # in units of 8 rows, and dense
def test_pages_outside_the_pool_and_lengths_beyond_the_table_stay_in_bounds(Hq, N):
    cache, table, held = small(L=200)
    q = rand((2, Hq, N, 128), 1, torch.bfloat16).to(DEV)
    good = gfa.attention_flash_gqa_kv4(q, cache, table, i32([200, 160]), causal=True)
    for page in (-1, cache.num_pages, 2 ** 31 - 1, -2 ** 31):
        bad = table.clone()
        bad[0, 2] = page
        o = gfa.attention_flash_gqa_kv4(q, cache, bad, i32([200, 160]), causal=True)
        assert status() == PAGE
        assert torch.equal(o[1], good[1])  # the other request is as it was
        gfa.kv4_read(cache, bad, i32([200, 160]), 200)
        assert status() == PAGE
    full = table.shape[1] * 16
    for n in (full + 1, 2 ** 31 - 1):
        o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([n, 160]), causal=True)
        assert status() == LENGTH
        assert torch.equal(o[1], good[1])
    o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([-5, 160]), causal=True, q_lens=i32([-3, N]))
    assert (o[0] == 0).all() and torch.equal(o[1], good[1])


# ------------------------------------------------------------------ masked places
@pytest.mark.parametrize("D", [64, 512])
@pytest.mark.parametrize("Hq,Hkv,N", [(4, 2, 2), (32, 4, 240)])  # in units of 8 rows, and dense
def test_non_finite_values_do_not_leave_the_rows_that_see_them(D, Hq, Hkv, N):
    """Tokens whose keys or values hold a NaN or an infinity: rows that see them are NaN in that group at
    least, the others are as if the tokens were not there."""
    B, L, page = 1, 300, 16
    G = Hq // Hkv
    cache = gfa.kv4_alloc(-(-L // page), Hkv, D, page, torch.bfloat16, DEV)
    table = scattered_table(B, -(-L // page), cache.num_pages, 1)
    k, v = (rand((B, Hkv, L, D), s, torch.bfloat16) for s in (1, 2))
    q = rand((B, Hq, N, D), 3, torch.bfloat16).to(DEV)
    last = L - 1  # seen by the last row only
    clean = {}
    for what in ("none", "key", "value"):
        kk, vv = k.clone(), v.clone()
        if what == "key":
            kk[0, 0, last, 5], kk[0, 1, last, D - 1] = math.nan, math.inf
        if what == "value":
            vv[0, 0, last, 5], vv[0, 1, last, D - 1] = -math.inf, math.nan
        gfa.kv4_append(cache, kk.to(DEV), vv.to(DEV), slots_of(table, [0], L, [L], page))
        o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([L]), causal=True)
        if what == "none":
            clean = o
            continue
        assert torch.equal(o[:, :, :-1], clean[:, :, :-1])
        for h in range(Hq):
            if h // G < 2:
                group = slice(0, 64) if h // G == 0 else slice(D - 64, D)
                assert torch.isnan(o[0, h, -1, group]).all()
            else:
                assert torch.equal(o[0, h, -1], clean[0, h, -1])
    # outside the window of the rows from position 110 on
    vv, kk = v.clone(), k.clone()
    vv[0, :, 10], kk[0, :, 10] = math.nan, math.inf
    gfa.kv4_append(cache, kk.to(DEV), vv.to(DEV), slots_of(table, [0], L, [L], page))
    o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([L]), causal=True, slide_size=100)
    sees = max(0, 110 - (L - N))
    assert torch.isnan(o[:, :, :sees]).all() and torch.isfinite(o[:, :, sees:]).all()


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.float16),
                                     (512, torch.bfloat16)], ids=ids)
@pytest.mark.parametrize("Hq,N", [(4, 2), (32, 240)])  # in units of 8 rows, and dense
@pytest.mark.parametrize("at", [0, 150, 298])
def test_a_nan_that_is_seen_with_hardly_any_weight_is_seen(D, dtype, Hq, N, at):
    """exp(-2 * 16 * sqrt(D)) is 0 in fp32 (the least is exp(-103)), but not in the formula: NaN times it is NaN."""
    Hkv, L = 4, 300
    cache = gfa.kv4_alloc(-(-L // 16), Hkv, D, 16, dtype, DEV)
    table = scattered_table(1, -(-L // 16), cache.num_pages, 1)
    k = torch.full((1, Hkv, L, D), 4.0, dtype=dtype)
    v = rand((1, Hkv, L, D), 2, dtype)
    k[:, :, at], v[:, :, at, 3] = -4.0, math.nan
    gfa.kv4_append(cache, k.to(DEV), v.to(DEV), slots_of(table, [0], L, [L], 16))
    q = torch.full((1, Hq, N, D), 4.0, dtype=dtype, device=DEV)
    o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([L]), causal=True)
    sees = torch.arange(L - N, L) >= at
    assert torch.isnan(o[0, :, sees, 3]).all()
    assert torch.isfinite(o[0, :, ~sees]).all()


@pytest.mark.parametrize("Hq", [4, 64])  # in units of 8 rows, and dense
def test_a_window_of_any_length(Hq):
    """Windows as long as the table and longer are none, also where rows lie before the first key."""
    cache, table, _ = small(L=200)
    lens, ql = i32([4, 200]), i32([40, 40])
    q = rand((2, Hq, 40, 128), 1, torch.bfloat16).to(DEV)
    want = gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True, q_lens=ql)
    for window in (table.shape[1] * 16, 2 ** 31 - 1):
        assert torch.equal(gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True, slide_size=window,
                                                       q_lens=ql), want)
    assert (want[0, :, :36] == 0).all() and (want[0, :, 36:] != 0).any()


@pytest.mark.parametrize("Hq,N", [(4, 1), (32, 150)])  # in units of 8 rows, and dense
def test_a_bound_that_does_not_hold_touches_one_request(Hq, N):
    cache, table, _ = small(L=200)
    q = rand((2, Hq, N, 128), 1, torch.bfloat16).to(DEV)
    good = gfa.attention_flash_gqa_kv4(q, cache, table, i32([200, 160]), causal=True)
    o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([200, 160]), causal=True, max_kv_len=160)
    assert torch.equal(o[1], good[1])
    assert status() == LENGTH or torch.equal(o, good)


def test_a_query_that_is_not_finite_spoils_its_row_only():
    cache, table, held = small(L=300)
    q = rand((2, 4, 3, 128), 1, torch.bfloat16).to(DEV)
    clean = gfa.attention_flash_gqa_kv4(q, cache, table, i32([300, 40]), causal=True)
    bad = q.clone()
    bad[0, 1, 1, 7], bad[1, 3, 0, 0] = math.inf, math.nan
    o = gfa.attention_flash_gqa_kv4(bad, cache, table, i32([300, 40]), causal=True)
    hit = torch.zeros(2, 4, 3, dtype=torch.bool, device=DEV)
    hit[0, 1, 1] = hit[1, 3, 0] = True
    assert torch.isnan(o[hit]).all() and torch.equal(o[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("factor", [1e-3, 300.0])
def test_values_far_from_one(dtype, factor):
    """Small and large keys and values: P' = scale * P keeps its range."""
    cache, table, held = filled(2, 2, 128, 900, 64, dtype, 5, factor)
    q = (rand((2, 4, 2, 128), 1, dtype) * min(1.0, 1 / factor)).to(DEV)
    check(q, cache, table, held, [900, 333], None, True, 0)


def test_one_large_score_among_many_small_ones():
    """The running maximum is raised late, by a lot, in one warp's block only."""
    L, D = 4000, 128
    k, v = rand((1, 1, L, D), 1, torch.bfloat16), rand((1, 1, L, D), 2, torch.bfloat16)
    q = rand((1, 8, 1, D), 3, torch.bfloat16)
    for at, gain in ((0, 30.0), (1777, 30.0), (3999, 60.0)):
        k[0, 0, at] = q[0, 3, 0] * gain
    cache = gfa.kv4_alloc(64, 1, D, 64, torch.bfloat16, DEV)
    table = scattered_table(1, 63, 64, 1)
    gfa.kv4_append(cache, k.to(DEV), v.to(DEV), slots_of(table, [0], L, [L], 64))
    held = [kv4_ref.values(*kv4_ref.quantise(x.to(DEV))) for x in (k, v)]
    check(q.to(DEV), cache, table, held, [L], None, True, 0)


# ------------------------------------------------------------------ tables, layouts, bounds
def test_requests_may_share_pages_and_tables_may_be_views():
    cache, table, held = small(L=400, B=1)
    both = torch.cat([table, table])[:, None].expand(2, 3, -1).reshape(6, -1)  # six requests on one prefix
    wide = torch.stack([both, both + 1], 1)[:, 0]                              # rows with a stride of their own
    q = rand((6, 4, 1, 128), 1, torch.bfloat16).to(DEV)
    lens = [400, 399, 16, 17, 1, 256]
    o, _ = check(q, cache, wide, [h.expand(6, -1, -1, -1) for h in held], lens, None, True, 0)
    same = gfa.attention_flash_gqa_kv4(q, cache, both.contiguous(), i32(lens), causal=True, max_kv_len=400)
    assert torch.equal(o, same)


def test_pages_behind_the_first_4_gib():
    """The same tokens in a small cache and in the last pages of one of 8.5 GiB."""
    Hkv, D, page, L, dtype = 4, 512, 256, 300, torch.bfloat16
    k, v = (rand((1, Hkv, L, D), s, dtype).to(DEV) for s in (1, 2))
    q = rand((1, 32, 130, D), 3, dtype).to(DEV)
    got = []
    for total, pages in ((2, [1, 0]), (16384, [16383, 8192])):
        cache = gfa.kv4_alloc(total, Hkv, D, page, dtype, DEV)
        table = i32([pages])
        gfa.kv4_append(cache, k, v, slots_of(table, [0], L, [L], page))
        got.append([*gfa.kv4_read(cache, table, i32([L]), L),
                    gfa.attention_flash_gqa_kv4(q, cache, table, i32([L]), causal=True),
                    gfa.attention_flash_gqa_kv4(q[:, :, :1], cache, table, i32([L]), causal=True)])
    assert cache.pages.numel() > 2 ** 33
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("Hq,N", [(4, 1), (32, 130)])  # in units of 8 rows, and dense
def test_query_layouts(Hq, N):
    cache, table, held = small(L=300)
    base = rand((2, N, Hq, 128), 1, torch.bfloat16).to(DEV)
    want = gfa.attention_flash_gqa_kv4(base.transpose(1, 2).contiguous(), cache, table, i32([300, 131]), causal=True)
    views = [base.transpose(1, 2), torch.cat([base, base], -1)[..., :128].transpose(1, 2),
             torch.nn.functional.pad(base, (4, 4))[..., 4:-4].transpose(1, 2)]
    for q in views:
        o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([300, 131]), causal=True)
        assert torch.equal(o, want)
    one = base[:, :, :1].transpose(1, 2)
    o = gfa.attention_flash_gqa_kv4(one.expand(2, Hq, N, 128), cache, table, i32([300, 131]), causal=True)
    o2 = gfa.attention_flash_gqa_kv4(one.repeat(1, Hq, 1, 1), cache, table, i32([300, 131]), causal=True)
    assert torch.equal(o, o2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_many_tokens_at_once_write_what_a_few_at_a_time_do(D, dtype):
    """Two lanes a group against four: groups of all magnitudes, ties at both ends, infinities and NaNs."""
    H, page = 8, 16
    N = 64000 * 64 // (H * D) + 37
    cols = -(-N // page)
    table = scattered_table(1, cols, cols, 5)
    slots = slots_of(table, [0], N, [N - 5], page)
    k, v = (rand((1, H, N, D), s, torch.float32) for s in (1, 2))
    top = 15 if dtype == torch.float16 else 126
    k = k * torch.exp2(torch.randint(-top, top, (1, 1, N, D // 64), generator=torch.Generator().manual_seed(3))
                       .float()).repeat_interleave(64, -1)
    v[:, :, ::3] = (v[:, :, ::3] * 4).round().clamp(-15, 15) / 2  # many ties
    v[:, :, ::7] = torch.where(v[:, :, ::7] > 0, 7.5, -7.5)       # both ends of the range
    k, v = k.to(dtype), v.to(dtype)
    v[0, 0, 11, 3], v[0, 1, 12, D - 1], k[0, 2, 13, D // 2] = math.nan, math.inf, -math.inf
    k, v = k.to(DEV), v.to(DEV)
    caches = [gfa.kv4_alloc(cols, H, D, page, dtype, DEV) for _ in range(2)]
    for c in caches:
        c.pages.fill_(0xA5)
    gfa.kv4_append(caches[0], k, v, slots)
    for i in range(0, N, 500):
        gfa.kv4_append(caches[1], k[:, :, i:i + 500], v[:, :, i:i + 500], slots[:, i:i + 500])
    assert torch.equal(caches[0].pages, caches[1].pages)
    got = gfa.kv4_read(caches[0], table, i32([N - 5]), 200)
    for x, y in zip(got, (k, v)):
        want = kv4_ref.values(*kv4_ref.quantise(y[:, :, :200]))
        assert torch.equal(torch.nan_to_num(x.double(), nan=1e300), torch.nan_to_num(want, nan=1e300))


def test_the_cache_is_outside_autograd():
    cache, table, _ = small(L=100)
    k = rand((2, 2, 3, 128), 1, torch.bfloat16).to(DEV)
    slots = i32([[0, 1, 2], [3, 4, -1]])
    gfa.kv4_append(cache, k, k, slots)
    want = cache.pages.clone()
    gfa.kv4_append(cache, torch.zeros_like(k), torch.zeros_like(k), slots)
    leaf = k.clone().requires_grad_()
    gfa.kv4_append(cache, leaf * 1, leaf, slots)
    assert torch.equal(cache.pages, want) and not cache.pages.requires_grad
    for t in gfa.kv4_read(cache, table, i32([100, 50]), 100):
        assert not t.requires_grad
    with pytest.raises(NotImplementedError, match="backward"):
        gfa.attention_flash_gqa_kv4(leaf, cache, table, i32([100, 50]))


@pytest.mark.parametrize("n", [1, 5, 100, 1000])  # one group a warp, and four
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_read_of_few_and_many_rows(D, n):
    B, H, L = 3, 7, 1000
    cache, table, held = filled(B, H, D, L, 64, torch.bfloat16, 9)
    lens, start = [L, 0, 37], [L - n, 0, 30]
    for i, t in enumerate(gfa.kv4_read(cache, table, i32(lens), n, starts=i32(start))):
        for b in range(B):
            want = torch.zeros(H, n, D, dtype=torch.float64, device=DEV)
            m = max(0, min(n, lens[b] - start[b]))
            want[:, :m] = held[i][b, :, start[b]:start[b] + m]
            assert torch.equal(t[b].double(), want)


def test_read_from_any_start():
    cache, table, held = small(L=200, B=3)
    lens, starts = [200, 64, 5], [33, 64, 0]
    k, v = gfa.kv4_read(cache, table, i32(lens), 90, starts=i32(starts))
    for got, want in ((k, held[0]), (v, held[1])):
        for b in range(3):
            n = max(0, min(90, lens[b] - starts[b]))
            assert torch.equal(got[b, :, :n].double(), want[b, :, starts[b]:starts[b] + n])
            assert (got[b, :, n:] == 0).all()


# ------------------------------------------------------------------ streams, graphs, workspaces
def test_calls_on_two_streams_at_once():
    cache, table, held = small(L=3000, D=256)
    qs = [rand((2, 8, n, 256), n, torch.bfloat16).to(DEV) for n in (1, 3, 1, 200)]
    lens = i32([3000, 1234])
    want = [gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(10):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_captured_calls_follow_lengths_that_change():
    cache, table, held = small(L=2000, D=64)
    q1, q2 = (rand((2, h, n, 64), n, torch.bfloat16).to(DEV) for h, n in ((4, 1), (32, 160)))
    lens, new = i32([10, 10]), i32([1, 1])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for q in (q1, q2):
            gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True, q_lens=new)
    torch.cuda.synchronize()
    graphs = []
    for q in (q1, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True, q_lens=new)
        graphs.append((g, out, q))
    for a, b, n in ((2000, 1, 1), (0, 777, 1), (1999, 2000, 0), (160, 16, 1)):
        lens.copy_(i32([a, b]))
        new.copy_(i32([n, 1]))
        for g, out, q in graphs:
            g.replay()
        for g, out, q in graphs:
            want = gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True, q_lens=new)
            assert torch.equal(out, want)


def test_two_runs_give_the_same_bits():
    cache, table, held = small(L=5000, D=512, page=64)
    q = rand((2, 8, 1, 512), 1, torch.bfloat16).to(DEV)
    first = gfa.attention_flash_gqa_kv4(q, cache, table, i32([5000, 4321]), causal=True)
    for _ in range(20):
        assert torch.equal(first, gfa.attention_flash_gqa_kv4(q, cache, table, i32([5000, 4321]), causal=True))


def test_a_chunk_and_its_tokens_alone_agree():
    """The dense path of a chunk and the 8-row units of its single tokens see the same cache."""
    cache, table, held = small(L=500)
    q = rand((2, 64, 64, 128), 1, torch.bfloat16).to(DEV)
    whole = gfa.attention_flash_gqa_kv4(q, cache, table, i32([500, 100]), causal=True)
    for at in (0, 17, 63):
        one = gfa.attention_flash_gqa_kv4(q[:, :, at:at + 1], cache, table, i32([500 - 63 + at, 100 - 63 + at]), causal=True)
        _, _, bound = kv4_ref.attention(q[:, :, at:at + 1], *held, [500 - 63 + at, 100 - 63 + at], [1, 1], True, 0, 128 ** -0.5)
        assert ((whole[:, :, at:at + 1].double() - one.double()).abs() <= 2 * bound).all()


def test_waits_time_out_and_the_next_call_is_correct():
    """No copy is issued, so every wait runs into its (short) bound; see test_timeout_gpu.py."""
    cache, table, held = small(L=700, D=256)
    q = rand((2, 4, 1, 256), 1, torch.bfloat16).to(DEV)
    lib = _lib.load()
    lib.gqafa_set_test_waits(2_000_000, 1)
    try:
        gfa.attention_flash_gqa_kv4(q, cache, table, i32([700, 300]), causal=True)
        assert status() in {1, 2, 3, 4, 5, 6}
    finally:
        lib.gqafa_set_test_waits(0, 0)
    check(q, cache, table, held, [700, 300], None, True, 0)
