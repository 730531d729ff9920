"""gqafa_kv4_attend called as a C program calls it, with a workspace of the size that
gqafa_kv4_attend_workspace_size gives for the documented arguments."""
import pytest
import torch

import gemma_triton_flash_attn as gfa
import kv4_ref
from gemma_triton_flash_attn import _lib
from test_kv4_gpu import DEV, filled, i32, rand

pytestmark = pytest.mark.gpu


def size_of(q, cache, max_kv_len, window):
    B, Hq, N, D = q.shape
    return _lib.load().gqafa_kv4_attend_workspace_size(B, Hq, cache.num_kv_heads, N, D, max_kv_len, window)


def attend(q, cache, table, lens, max_kv_len, causal, window, workspace_bytes):
    """Return code, O: the workspace is filled with NaNs and followed by bytes that must stay."""
    B, Hq, N, D = q.shape
    ws = torch.full((workspace_bytes + 4096,), 0xFF, dtype=torch.uint8, device=DEV)
    o = torch.full_like(q, 7.0)
    rc = _lib.load().gqafa_kv4_attend(
        q.data_ptr(), _lib.strides_arg(q.stride()), cache.pages.data_ptr(), cache.num_pages, table.data_ptr(),
        table.stride(0), table.shape[1], lens.data_ptr(), None, o.data_ptr(), _lib.strides_arg(o.stride()), None, B, Hq,
        cache.num_kv_heads, N, D, cache.page_size, max_kv_len, D ** -0.5, int(causal), window, 1, ws.data_ptr(),
        workspace_bytes, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (ws[workspace_bytes:] == 0xFF).all()
    return rc, o


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("B,Hq,Hkv,N,L", [(2, 8, 4, 1, 5000), (1, 32, 4, 1, 9400), (2, 64, 4, 140, 700),
                                          (1, 64, 4, 140, 4700)])  # units of 8 rows, and dense
@pytest.mark.parametrize("what", ["exact", "zero", "above", "window"])
def test_workspaces_of_the_documented_size_are_enough(B, Hq, Hkv, N, L, what, D):
    cache, table, held = filled(B, Hkv, D, L, 64, torch.bfloat16, 4)
    q = rand((B, Hq, N, D), 2, torch.bfloat16).to(DEV)
    lens, capacity = [L, L // 3][:B], table.shape[1] * 64
    causal, window, max_kv_len = True, 0, capacity
    size = size_of(q, cache, capacity, 0)
    if what == "zero":  # the table's capacity
        max_kv_len, size = 0, size_of(q, cache, 0, 0)
    if what == "above":  # a bound that the table's capacity undercuts
        bounds = [capacity + 1, capacity + 200, 2 * capacity, 8 * capacity, 1 << 20]
        sizes = [size_of(q, cache, n, 0) for n in bounds]
        assert sizes == sorted(sizes)
        max_kv_len, size = bounds[1], sizes[1]
    if what == "window":  # which counts only with causal
        causal, window, size = False, 100, size_of(q, cache, capacity, 100)
    assert size > 0
    rc, o = attend(q, cache, table, i32(lens), max_kv_len, causal, window, size)
    assert rc == _lib.GQAFA_OK, _lib.load().gqafa_last_error()
    want, _, bound = kv4_ref.attention(q, *held, lens, [N] * B, causal, 0, D ** -0.5)
    assert ((o.double() - want).abs() <= bound).all()
    if what in ("exact", "above"):
        same = gfa.attention_flash_gqa_kv4(q, cache, table, i32(lens), causal=causal)
        assert torch.equal(o, same)
    assert _lib.device_status(torch.cuda.current_device(), reset=True) == 0


@pytest.mark.parametrize("N", [1, 140])
def test_a_workspace_that_is_too_small_is_refused(N):
    cache, table, _ = filled(1, 4, 128, 5000, 64, torch.bfloat16, 4)
    q = rand((1, 64, N, 128), 2, torch.bfloat16).to(DEV)
    for size in (0, 256, 4096):
        rc, o = attend(q, cache, table, i32([5000]), 0, True, 0, size)
        assert rc == _lib.GQAFA_ERR_INVALID and b"workspace" in _lib.load().gqafa_last_error()
        assert (o == 7).all()


def test_size_call_refuses_what_the_launch_refuses():
    size = _lib.load().gqafa_kv4_attend_workspace_size
    assert size(1, 8, 3, 1, 128, 100, 0) == -1 and size(1, 8, 4, 1, 96, 100, 0) == -1
    assert size(1, 8, 4, 1, 128, -1, 0) == -1 and size(1, 8, 4, 1, 128, 100, -1) == -1


@pytest.mark.parametrize("B,Hq,Hkv,N,dense", [(6, 8, 8, 64, False), (6, 32, 4, 200, True)])
def test_requests_that_are_written_out_one_at_a_time_count_a_launch_each(B, Hq, Hkv, N, dense):
    """A table for 131072 tokens, head_dim 512: one request or two fill the 2 GiB, so six requests are several
    launches of a wave each, which a few rows are not worth."""
    D, capacity, lens = 512, 131072, [600, 240, 64, 0, 257, 333]
    cache, table, held = filled(B, Hkv, D, 600, 64, torch.bfloat16, 31)
    wide = torch.full((B, capacity // 64), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = rand((B, Hq, N, D), 8, torch.bfloat16).to(DEV)
    assert (size_of(q, cache, capacity, 0) >= 2 ** 30) == dense
    assert (size_of(q, cache, 1024, 0) >= 2 ** 24) == (N >= 64)  # a short table: all in one launch
    o = gfa.attention_flash_gqa_kv4(q, cache, wide, i32(lens), causal=True)
    want, _, bound = kv4_ref.attention(q, *held, lens, [N] * B, True, 0, D ** -0.5)
    assert ((o.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("D", [128, 512])
@pytest.mark.parametrize("fits", [1, 2, 3])
def test_a_workspace_for_fewer_requests_at_a_time_gives_the_same_bits(fits, D):
    """Groups of one and two requests of three, with a NaN in a value group of each."""
    B, Hq, Hkv, N, L = 3, 32, 4, 200, 600
    cache, table, _ = filled(B, Hkv, D, L, 64, torch.bfloat16, 4)
    bad = rand((B, Hkv, 1, D), 5, torch.bfloat16).to(DEV)
    bad[0, 1, 0, 5], bad[1, 2, 0, D - 1], bad[2, 0, 0, 64] = float("nan"), float("inf"), -float("inf")
    page = table[:, 400 // 64].tolist()
    gfa.kv4_append(cache, bad, bad.nan_to_num(0, 0, 0), i32([[p * 64 + 400 % 64] for p in page]))  # keys first
    gfa.kv4_append(cache, bad.nan_to_num(0, 0, 0), bad, i32([[p * 64 + 400 % 64] for p in page]))
    q, lens = rand((B, Hq, N, D), 2, torch.bfloat16).to(DEV), i32([L, 450, 590])
    want = gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True)
    assert torch.isnan(want).any() and torch.isfinite(want).any()
    capacity = table.shape[1] * 64
    whole = size_of(q, cache, capacity, 0)
    one = Hkv * capacity * (4 * D + D / 512)  # K, V and a bit for each token and group
    assert whole == 3 * one
    rc, o = attend(q, cache, table, lens, capacity, True, 0, int(one) * fits)
    assert rc == _lib.GQAFA_OK
    assert torch.equal(o.nan_to_num(1e9), want.nan_to_num(1e9)) and torch.equal(torch.isnan(o), torch.isnan(want))


def test_groups_that_are_too_small_to_pay_are_not_made():
    """24 requests whose keys and values fit the workspace one at a time: units of 8 rows, as the same call with
    max_kv_len 0 in the size call; and no workspace, or a negative size, is refused."""
    B, Hq, Hkv, N, D, L = 24, 8, 4, 48, 128, 300
    cache, table, held = filled(B, Hkv, D, L, 64, torch.bfloat16, 4)
    q, lens = rand((B, Hq, N, D), 2, torch.bfloat16).to(DEV), i32([L] * B)
    capacity = table.shape[1] * 64
    units = size_of(q, cache, 0, 0)
    one = Hkv * capacity * (4 * D + D // 512)
    assert size_of(q, cache, capacity, 0) > units > one
    rc, o = attend(q, cache, table, lens, capacity, True, 0, units)
    rc0, o0 = attend(q, cache, table, lens, 0, True, 0, units)
    assert rc == rc0 == _lib.GQAFA_OK and torch.equal(o, o0)
    dense = gfa.attention_flash_gqa_kv4(q, cache, table, lens, causal=True)
    want, _, bound = kv4_ref.attention(q, *held, [L] * B, [N] * B, True, 0, D ** -0.5)
    for got in (o, dense):
        assert ((got.double() - want).abs() <= bound).all()
    for bad in (0, -1, -2 ** 40):
        lib = _lib.load()
        rc = lib.gqafa_kv4_attend(
            q.data_ptr(), _lib.strides_arg(q.stride()), cache.pages.data_ptr(), cache.num_pages, table.data_ptr(),
            table.stride(0), table.shape[1], lens.data_ptr(), None, o.data_ptr(), _lib.strides_arg(o.stride()), None, B,
            Hq, Hkv, N, D, cache.page_size, capacity, D ** -0.5, 1, 0, 1, dense.data_ptr(), bad,
            torch.cuda.current_stream().cuda_stream)
        assert rc == _lib.GQAFA_ERR_INVALID and b"workspace" in lib.gqafa_last_error()
