"""How exactly the paged 4-bit cache's attention computes, where a coarse bound would hide an error: weights
far below the largest one, values of any magnitude.

The tests here use queries whose 16-bit integers are exact (multiples of 1/32 up to 127/32, the largest one
in every group), and a bound that goes with the values' size: an output of zeros does not pass."""
import math

import pytest
import torch

import gemma_triton_flash_attn as gfa
import kv4_ref
from gemma_triton_flash_attn import _lib
from test_kv4_gpu import DEV, i32, ids, rand, scattered_table, slots_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.device_status(torch.cuda.current_device(), reset=True)
    yield
    assert _lib.device_status(torch.cuda.current_device(), reset=True) == 0, "a kernel recorded a status"


def exact_query(shape, seed, dtype):
    """Multiples of 1/32 between -127/32 and 127/32, 127/32 among every 64: 32512 / max|q| = 8192 is exact."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, shape, generator=g).float()
    q[..., ::64] = 127
    return (q / 32).to(dtype).to(DEV)


def cache_of(k, v, page=64, seed=1):
    """A cache that holds k and v (B, H, L, D) whole, and its table; stale slots hold anything."""
    B, H, L, D = k.shape
    cols = -(-L // page)
    cache = gfa.kv4_alloc(B * cols + 1, H, D, page, k.dtype, DEV)
    cache.pages.random_(0, 256, generator=torch.Generator(DEV).manual_seed(seed))
    table = scattered_table(B, cols, B * cols + 1, seed)
    gfa.kv4_append(cache, k.to(DEV), v.to(DEV), slots_of(table, [0] * B, L, [L] * B, page))
    return cache, table


def attend64(q, k, v, lens, causal=True, window=0):
    """O and an element-wise bound in float64 over the values that a cache of k and v (16 bits) holds, for
    queries as exact_query gives them, N rows that are each request's last positions.

    Roundings, to first order (u: half a step of the 16-bit type, e = 2^-23):
      output   u |O|, and half a step of the type's smallest numbers;
      s * P    u per key where it is a normal number: 1.01 u sum_j P_j |v_j|. fp16: below 2^-14 it is off by up to
               2^-25, of P >= 2^-3 for the largest weight and the head's largest scale brought to at least 2^13: a
               key's part of the output by at most 15 * 2^-25 * 2^-13 * 2^3 of that scale (units of 8 rows);
      scores   fp32 sums of integers, D / 64 terms s * (integer part) and their products: (D / 64 + 4) e of
               scale * 31 * sum_d |q_d| s, and P by twice that, relative;
      sums     up to 8 MMA steps of a tile, of terms up to (256 + 15) s P, twice (products and offsets); then one
               addition a tile (128 keys or more, 64 parts at most) of terms up to 15 s P, half of e each;
      exp2 and the joins of parts: 16 steps of fp32 relative to P."""
    B, Hq, N, D = q.shape
    G = Hq // k.shape[1]
    u, e = kv4_ref.ROUND[q.dtype], 2.0 ** -23
    O = torch.zeros(B, Hq, N, D, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(O)
    for b in range(B):
        L = lens[b]
        kc, ks, kz = kv4_ref.quantise(k[b, :, :L].to(DEV))
        vc, vs, vz = kv4_ref.quantise(v[b, :, :L].to(DEV))
        kk, vv = (kv4_ref.values(*x).repeat_interleave(G, 0) for x in ((kc, ks, kz), (vc, vs, vz)))
        kstep, vstep = (x.repeat_interleave(64, -1).repeat_interleave(G, 0) for x in (ks, vs))
        pos, key = L - N + torch.arange(N, device=DEV)[:, None], torch.arange(L, device=DEV)[None]
        ok = (key <= pos) & (key > pos - (window or L + N)) if causal else torch.ones(N, L, dtype=torch.bool, device=DEV)
        qq = q[b].double()
        s = (qq @ kk.transpose(-1, -2) * D ** -0.5).masked_fill(~ok, -math.inf)
        off = (D / 64 + 4) * e * D ** -0.5 * 31 * (qq.abs() @ kstep.transpose(-1, -2))
        off = off.masked_fill(~ok, 0).amax(-1, keepdim=True) + 16 * e
        p = torch.softmax(s, -1)
        o, size, steps = p @ vv, p @ vv.abs(), p @ vstep
        O[b] = o
        bound[b] = (u * o.abs() + 1.01 * u * size + 2 * off * size
                    + e * (2 * 8 * 271 + (L / 128 + 64) * 15 / 2) * steps
                    + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2)
        if q.dtype == torch.float16:
            seen = ok.double().sum(-1)[:, None]
            bound[b] += seen * 15 * 2.0 ** -35 * vstep.amax((-2, -1), keepdim=True)
    return O, bound


def compare(q, k, v, lens=None, causal=True, window=0, page=64):
    cache, table = cache_of(k, v, page)
    lens = [k.shape[2]] * k.shape[0] if lens is None else lens
    o = gfa.attention_flash_gqa_kv4(q, cache, table, i32(lens), causal=causal, slide_size=window)
    want, bound = attend64(q, k, v, lens, causal, window)
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all()
    assert (err <= bound).all(), f"error {err.max():.3e} of {want.abs().max():.3e}, {(err / bound).max():.2f} bounds"
    return o, want, bound


# ------------------------------------------------------------------ weights of many magnitudes
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("D,L,sink,size", [(128, 16384, 9.7, 0.02), (64, 131072, 12.0, 0.1), (512, 16384, 9.7, 1e-3),
                                           (256, 4096, 0.0, 1e-4), (128, 4096, 5.0, 3000.0)])
def test_small_weights_count_whatever_the_values_size(D, L, sink, size, dtype):
    """One key with a far larger score than the others, which together weigh as much or more."""
    Hq = 8
    q = exact_query((1, Hq, 1, D), 1, dtype)
    rows = q[0, :, 0].float().cpu()
    k = 0.3 * torch.randn(1, 1, L, D, generator=torch.Generator().manual_seed(2)) * D ** 0.5 / rows.norm(dim=1).mean() * 2
    k[0, 0, 0] = (rows / rows.norm(dim=1, keepdim=True) ** 2).sum(0) * sink * D ** 0.5
    v = size * (1 + 0.3 * torch.randn(1, 1, L, D, generator=torch.Generator().manual_seed(3)))
    _, want, bound = compare(q, k.to(dtype), v.to(dtype))
    assert (want.abs() > 10 * bound).double().mean() > 0.99  # zeros would fail


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("D,Hq,N,L", [(64, 4, 1, 3000), (128, 8, 5, 700), (256, 8, 1, 20000), (512, 16, 1, 9000),
                                      (128, 32, 150, 600)])  # the last one on the dense path
def test_values_times_a_power_of_two_give_outputs_times_it(D, Hq, N, L, dtype):
    k, v = rand((2, 2, L, D), 1, dtype), (rand((2, 2, L, D), 2, torch.float32) + 1).to(dtype)
    q = rand((2, Hq, N, D), 3, dtype).to(DEV)
    got = []
    for power in (0, -6, 5):
        cache, table = cache_of(k, (v.float() * 2.0 ** power).to(dtype))
        o = gfa.attention_flash_gqa_kv4(q, cache, table, i32([L, L // 2]), causal=True)
        got.append((o.double() * 2.0 ** -power, 2.0 ** power))
    least = 2 * torch.finfo(dtype).smallest_normal
    for o, factor in got[1:]:
        normal = got[0][0].abs() * factor > least
        assert normal.double().mean() > 0.9
        assert torch.equal(o[normal], got[0][0][normal])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("order", ["up", "down", "mixed", "late"])
def test_values_whose_size_changes_along_the_cache(D, order, dtype):
    """The scales that a unit meets rise, fall, jump, or rise at the very end."""
    L, N = 2500, 2
    at = torch.linspace(-9, 9, L)
    power = {"up": at, "down": -at, "mixed": at[torch.randperm(L, generator=torch.Generator().manual_seed(5))],
             "late": torch.where(torch.arange(L) < L - 3, -9.0, 9.0)}[order].round()
    v = rand((2, 2, L, D), 2, torch.float32) * torch.exp2(power)[:, None]
    q = exact_query((2, 8, N, D), 3, dtype)
    k = rand((2, 2, L, D), 4, dtype, 0.5)
    compare(q, k, v.to(dtype), [L, 1300])
    compare(q, k, v.to(dtype), [L, 1300], window=700, page=16)


@pytest.mark.parametrize("D", [64, 512])
def test_fp16_values_over_the_whole_range_under_growing_scores(D):
    """Groups from -65504 to 65504 (scale 9216), with scores that grow by less than what raises the reference
    of the softmax, and by more."""
    L = 3000
    v = (torch.rand(1, 1, L, D, generator=torch.Generator().manual_seed(1)) * 2 - 1) * 65504
    v[..., ::64], v[..., 1::64] = 65504, -65504
    q = exact_query((1, 4, 1, D), 2, torch.float16)
    unit = q[0, 0, 0].float().cpu()
    unit = unit / unit.norm() ** 2 * D ** 0.5  # score 1 for the first head
    for step in (3.3 / 2500, 3.46 / 1500, 3.6 / 1000, 0.02):  # 5 in log2 units is 3.4657 in score
        k = (torch.arange(L) * step).clamp(max=40.0)[None, None, :, None] * unit
        compare(q, k.half(), v.half())


# ------------------------------------------------------------------ queries
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("large", [4, 64, 8192])
def test_one_large_channel_of_the_query_costs_the_others_nothing(D, large, dtype):
    """A channel that the keys do not use is 1, 16 and 2048 times the next largest one: multiples of 1/32
    next to 127/32 * large / 4 are exact in 24 bits."""
    for L, N, Hq in ((17, 1, 8), (1000, 3, 6)):
        q = exact_query((2, Hq, N, D), 1, dtype)
        q[0, :, :, 5] = 127 / 32 * large / 4
        q[1, ::2, :, D - 3] = -127 / 32 * large / 4
        k, v = rand((2, 2, L, D), 2, dtype), rand((2, 2, L, D), 3, dtype)
        k[..., 5], k[..., D - 3] = 0, 0
        compare(q, k, v, [L, L // 2 + 3])


def test_a_row_does_not_depend_on_the_rows_beside_it():
    """Rows with a large channel, zeros and NaNs among the eight rows of a unit."""
    L, D, dtype = 900, 128, torch.bfloat16
    k, v = rand((1, 1, L, D), 1, dtype), rand((1, 1, L, D), 2, dtype)
    cache, table = cache_of(k, v)
    q = rand((1, 8, 1, D), 3, dtype).to(DEV)
    want = gfa.attention_flash_gqa_kv4(q, cache, table, i32([L]), causal=True)
    other = q.clone()
    other[0, 1, 0, 7], other[0, 2], other[0, 5, 0, 0], other[0, 6, 0, 1] = 1e5, 0, math.nan, math.inf
    got = gfa.attention_flash_gqa_kv4(other, cache, table, i32([L]), causal=True)
    for h in (0, 3, 4, 7):
        assert torch.equal(got[0, h], want[0, h])
    assert torch.isfinite(got[0, 1:3]).all() and torch.isnan(got[0, 5:7]).all()


@pytest.mark.parametrize("D,Hq,N,L", [(64, 4, 1, 3000), (512, 16, 1, 9000), (128, 32, 150, 600)])
def test_bf16_keys_and_values_up_to_2_to_the_95(D, Hq, N, L):
    """Queries times 2^-90 and keys times 2^90 give the same scores."""
    dtype = torch.bfloat16
    k, v = rand((1, 2, L, D), 1, dtype), rand((1, 2, L, D), 2, dtype)
    q = rand((1, Hq, N, D), 3, dtype).to(DEV)
    got = []
    for pq, pk, pv in ((0, 0, 0), (-90, 90, 0), (0, 0, 92), (20, -20, -90)):
        cache, table = cache_of(k * 2.0 ** pk, v * 2.0 ** pv)
        o = gfa.attention_flash_gqa_kv4(q * 2.0 ** pq, cache, table, i32([L]), causal=True)
        got.append(o.double() * 2.0 ** -pv)
    for o in got[1:]:
        assert torch.equal(o, got[0])


def test_queries_too_small_for_a_reciprocal():
    """32512 / max|q| passes fp32's range below 2^-113: the query's integers are then fewer, not wrong."""
    L, D, dtype = 500, 128, torch.bfloat16
    k, v = rand((1, 1, L, D), 1, dtype), rand((1, 1, L, D), 2, dtype)
    q = rand((1, 8, 1, D), 3, dtype).to(DEV)
    got = []
    for pq, pk, factor in ((0, 0, 1.0), (-115, 90, 2.0 ** 25)):
        cache, table = cache_of(k * 2.0 ** pk, v)
        got.append(gfa.attention_flash_gqa_kv4(q * 2.0 ** pq, cache, table, i32([L]), causal=True,
                                               softmax_scale=factor * D ** -0.5).double())
    # steps of 1e-38 on queries of 2^-115: a score off by at most D^-0.5 * 2^24 * 1e-38 * sum |k| < 1e-2
    assert (got[1] - got[0]).abs().max() <= 2 * 1e-2 * v.double().abs().max()
    assert got[0].abs().max() > 0.1


def test_an_all_zero_query_weighs_every_key_alike():
    L, D = 333, 256
    for dtype in (torch.bfloat16, torch.float16):
        k, v = rand((1, 2, L, D), 1, dtype), rand((1, 2, L, D), 2, dtype)
        compare(torch.zeros(1, 4, 2, D, dtype=dtype, device=DEV), k, v)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("value", [0.0, 1.0, -0.37])
def test_constant_values_come_back(D, value, dtype):
    """The offset of the codes cancels: zeros are exactly zeros, whatever the weights."""
    L = 3001
    k, v = rand((1, 2, L, D), 1, dtype, 2.0), torch.full((1, 2, L, D), value, dtype=dtype)
    q = exact_query((1, 8, 3, D), 3, dtype)
    o, want, _ = compare(q, k, v)
    if value == 0:
        assert (o == 0).all()
    assert (want - want.flatten()[0]).abs().max() < 1e-12


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
def test_groups_of_very_different_size_in_one_head(dtype):
    """One dim group a thousand times the other, either way round, and rows of one token."""
    L, D = 2000, 128
    k, q = rand((2, 1, L, D), 1, dtype), exact_query((2, 8, 1, D), 2, dtype)
    v = 1 + 0.5 * rand((2, 1, L, D), 3, torch.float32)
    v[0, ..., :64] *= 2.0 ** -10
    v[1, ..., 64:] *= 2.0 ** 9
    compare(q, k, v.to(dtype), [L, 1])
    compare(q, k, v.to(dtype), [1, L])
