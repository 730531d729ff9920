"""What a NaN (or an infinity, which is held as one) in the paged 4-bit cache does to the attention's results:
the same in units of 8 rows and on the dense path, and what the formula says."""
import math

import pytest
import torch

import gemma_triton_flash_attn as gfa
from gemma_triton_flash_attn import _lib
from test_kv4_gpu import DEV, i32, ids, rand, scattered_table, slots_of

pytestmark = pytest.mark.gpu
PATHS = [(8, 2, 3), (32, 4, 240)]  # H_Q, H_KV, N: in units of 8 rows, and dense


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.device_status(torch.cuda.current_device(), reset=True)
    yield
    assert _lib.device_status(torch.cuda.current_device(), reset=True) == 0, "a kernel recorded a status"


def run(k, v, q, lens, q_lens, causal, window, page=16):
    B, H, L, D = k.shape
    cols = -(-L // page)
    cache = gfa.kv4_alloc(B * cols, H, D, page, k.dtype, DEV)
    cache.pages.random_(0, 256, generator=torch.Generator(DEV).manual_seed(3))
    table = scattered_table(B, cols, B * cols, 1)
    gfa.kv4_append(cache, k.to(DEV), v.to(DEV), slots_of(table, [0] * B, L, lens, page))
    return gfa.attention_flash_gqa_kv4(q, cache, table, i32(lens), causal=causal, slide_size=window,
                                       q_lens=i32(q_lens), return_lse=True)


def sees(b, lens, q_lens, N, causal, window, at):
    """Rows of request b that see the key at position `at`."""
    row = torch.arange(N, device=DEV)
    pos = lens[b] - q_lens[b] + row
    ok = (row < q_lens[b]) & (at < lens[b])
    if causal:
        ok &= at <= pos
        if window:
            ok &= at > pos - window
    return ok


CASES = [(True, 0), (True, 37), (False, 0)]


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16),
                                     (512, torch.bfloat16), (512, torch.float16)], ids=ids)
@pytest.mark.parametrize("Hq,Hkv,N", PATHS)
@pytest.mark.parametrize("causal,window", CASES)
def test_a_key_that_is_not_finite_leaves_no_finite_weights(D, dtype, Hq, Hkv, N, causal, window):
    """O and LSE of the rows that see it are NaN, the LSE is not that of a row that sees no key."""
    B, L, lens, q_lens = 2, 500, [500, 261], [N, N - 2]
    k, v = rand((B, Hkv, L, D), 1, dtype), rand((B, Hkv, L, D), 2, dtype)
    q = rand((B, Hq, N, D), 3, dtype).to(DEV)
    clean, clean_lse = run(k, v, q, lens, q_lens, causal, window)
    at = lens[0] - N // 2 - 1
    k[0, 1, at, D - 1] = math.inf
    o, lse = run(k, v, q, lens, q_lens, causal, window)
    G = Hq // Hkv
    hit = torch.zeros_like(lse, dtype=torch.bool)
    hit[0, G:2 * G] = sees(0, lens, q_lens, N, causal, window, at)
    assert hit.any()
    assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(o[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16),
                                     (512, torch.bfloat16), (512, torch.float16)], ids=ids)
@pytest.mark.parametrize("Hq,Hkv,N", PATHS)
@pytest.mark.parametrize("causal,window", CASES)
def test_a_value_group_that_is_not_finite_spoils_its_dims_only(D, dtype, Hq, Hkv, N, causal, window):
    """P * NaN in the 64 dims of the group, in the rows that see the token; all else as if it were finite."""
    B, L, lens, q_lens = 2, 500, [500, 261], [N, N - 2]
    G, NG = Hq // Hkv, D // 64
    k, v = rand((B, Hkv, L, D), 1, dtype), rand((B, Hkv, L, D), 2, dtype)
    q = rand((B, Hq, N, D), 3, dtype).to(DEV)
    clean, clean_lse = run(k, v, q, lens, q_lens, causal, window)
    # the first token, one in the middle, a page's last, one that a single row sees, one behind the last
    marks = [(0, 0, 0, 0), (0, 1, lens[0] - N // 2 - 1, NG - 1), (1, 0, 239, NG // 2), (1, 1, lens[1] - 1, 0),
             (1, 1, 262, 0)]
    hit = torch.zeros_like(clean, dtype=torch.bool)
    for b, h, at, g in marks:
        v[b, h, at, 64 * g + at % 64] = (math.nan, math.inf, -math.inf)[at % 3]
        rows = sees(b, lens, q_lens, N, causal, window, at)
        hit[b, h * G:(h + 1) * G, :, 64 * g:64 * g + 64] |= rows[None, :, None]
    assert hit.any() and not hit.all()
    o, lse = run(k, v, q, lens, q_lens, causal, window)
    assert torch.equal(torch.isnan(o), hit)
    assert torch.equal(lse, clean_lse)
    if dtype == torch.bfloat16:
        assert torch.equal(o[~hit], clean[~hit])
    else:  # a group's scale that no longer counts may move the power of two that the weights carry
        assert (o[~hit] - clean[~hit]).abs().max() <= 2 ** -10 * clean.abs().max()


@pytest.mark.parametrize("Hq,Hkv,N", PATHS)
def test_a_row_sees_the_same_nans_in_a_chunk_and_alone(Hq, Hkv, N):
    B, L, D, dtype = 1, 400, 256, torch.bfloat16
    k, v = rand((B, Hkv, L, D), 1, dtype), rand((B, Hkv, L, D), 2, dtype)
    for at in range(3, L, 29):
        v[0, at % Hkv, at, at % D] = math.nan
    q = rand((B, Hq, N, D), 3, dtype).to(DEV)
    o, _ = run(k, v, q, [L], [N], True, 25)
    for row in (0, 1, N - 1):
        one, _ = run(k, v, q[:, :, row:row + 1], [L - N + 1 + row], [1], True, 25)
        assert torch.equal(torch.isnan(one), torch.isnan(o[:, :, row:row + 1]))


def test_nans_go_to_the_rows_of_a_strided_output():
    """Queries (and outputs) as a projection leaves them, (B, N, H, D) in memory."""
    B, Hq, Hkv, N, L, D, dtype = 2, 32, 4, 160, 300, 128, torch.bfloat16
    k, v = rand((B, Hkv, L, D), 1, dtype), rand((B, Hkv, L, D), 2, dtype)
    v[0, 2, 200, 70], v[1, 3, 250, 1] = math.nan, math.inf
    base = rand((B, N, Hq, D), 3, dtype).to(DEV)
    for causal, window in CASES:
        want, _ = run(k, v, base.transpose(1, 2).contiguous(), [L, 299], [N, 100], causal, window)
        o, _ = run(k, v, base.transpose(1, 2), [L, 299], [N, 100], causal, window)
        assert o.stride() == base.transpose(1, 2).stride() and torch.isnan(o).any()
        assert torch.equal(torch.isnan(o), torch.isnan(want)) and torch.equal(o.nan_to_num(0), want.nan_to_num(0))
