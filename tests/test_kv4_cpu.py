"""The paged 4-bit KV cache without a GPU: the number format's own properties, shapes through the Meta
kernels, and the refusals of the Python layer and of the C ABI."""
import ctypes
import math

import numpy as np
import pytest
import torch

import gemma_triton_flash_attn as gfa
import kv4_ref
from gemma_triton_flash_attn import _lib


# ------------------------------------------------------------------ the format
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_held_values_are_exact_in_16_bits_and_within_a_step(dtype):
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(500, 128, generator=g) * torch.exp2(torch.randint(-10, 10, (500, 1), generator=g).float())).to(dtype)
    x[0], x[1, :64], x[2] = 0, 5.0, x[2].abs()
    c, s, z = kv4_ref.quantise(x)
    held = kv4_ref.values(c, s, z)
    assert torch.equal(held.to(dtype).double(), held)
    assert ((c >= 0) & (c <= 15)).all() and ((z >= 0) & (z <= 15)).all()
    m, _ = torch.frexp(s)
    assert torch.equal(m * 16, torch.round(m * 16))  # 4 significant bits
    err = (held - x.double()).abs().unflatten(-1, (-1, 64)).amax(-1)
    assert (err <= s).all()
    # half a step for almost all: only the top code can be cut, by the zero point's rounding
    off = ((held - x.double()).abs().unflatten(-1, (-1, 64)) > s[..., None] / 2)
    assert (off <= (c.unflatten(-1, (-1, 64)) == 15)).all()
    assert (held[0] == 0).all()


def test_pages_unpack_to_what_the_layout_says():
    """One word of keys and one of values placed by hand."""
    pages = np.zeros((2, 2, 1, 1, 2 * 544), np.uint8)  # head_dim 128, page_size 16
    r, j, grp = 13, 5, 1  # token 13 of page 1, dims 64 + 40 .. 64 + 47
    key = grp * 512 + ((r % 8) * 4 + j // 2) * 16 + (r // 8) * 8 + (j % 2) * 4
    pages[1, 0, 0, 0, key:key + 4] = np.array([0x75316420], "<u4").view(np.uint8)  # dims in order: 0 .. 7
    t = (r % 8) // 2
    val = grp * 512 + (t * 8 + (j ^ (2 * t))) * 16 + ((r // 8) * 2 + r % 2) * 4
    pages[1, 1, 0, 0, val:val + 4] = np.array([0x76543210], "<u4").view(np.uint8)
    one = np.array([0x3F80 | 3], "<u2").view(np.uint8)  # scale 1, zero point 3
    at = 2 * 512 + grp * 32
    pages[1, 0, 0, 0, at + 2 * ((r % 8) * 2 + r // 8):][:2] = one
    pages[1, 1, 0, 0, at + 2 * (t * 4 + (r // 8) * 2 + r % 2):][:2] = one
    held = kv4_ref.unpack(torch.from_numpy(pages), 1, 128, 16)
    for kind in range(2):
        assert held[16 + r, kind, 0, 64 + 40:64 + 48].tolist() == [-3, -2, -1, 0, 1, 2, 3, 4]
    held[16 + r, :, 0, 64 + 40:64 + 48] = 0
    others = np.delete(held[16 + r, :, 0, 64:], np.s_[40:48], axis=1)  # the group's other codes are 0: 0 - 3
    assert (others == -3).all()
    held[16 + r, :, 0, 64:] = 0
    assert (held == 0).all()


# ------------------------------------------------------------------ shapes
def test_meta_kernels_give_the_shapes():
    ops = _lib.ops()
    i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device="meta")  # noqa: E731
    out = ops.kv4_plan(i32(5), i32(5), i32(5, 9), i32(40), i32(2), 64, 7)
    assert [tuple(t.shape) for t in out] == [(5, 9), (5,), (5,), (5, 7), (5, 7), (2,), (5,)]
    assert all(t.dtype == torch.int32 for t in out)
    pages = torch.empty(11, 2, 3, 4, 2 * 544, dtype=torch.uint8, device="meta")
    k = torch.empty(5, 3, 7, 128, dtype=torch.float16, device="meta")
    assert ops.kv4_append(pages, k, k, i32(5, 7), 64) is None
    rk, rv = ops.kv4_read(pages, i32(5, 9), i32(5), 20, None, 64, torch.float16)
    assert rk.shape == rv.shape == (5, 3, 20, 128) and rk.dtype == torch.float16
    q = torch.empty(5, 12, 2, 128, dtype=torch.float16, device="meta")
    o, lse = ops.kv4_attend(q, pages, i32(5, 9), i32(5), None, 64, 0, True, 0, 0.1, True)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (5, 12, 2) and lse.dtype == torch.float32


# ------------------------------------------------------------------ refusals
def pages_of(n=4, heads=2, dim=128, page=64):
    return torch.zeros(n, 2, heads, page // 16, dim // 64 * 544, dtype=torch.uint8)


@pytest.mark.parametrize("kw,error", [
    (dict(head_dim=96), NotImplementedError), (dict(page_size=48), NotImplementedError),
    (dict(page_size=512), NotImplementedError), (dict(dtype=torch.float32), NotImplementedError),
    (dict(page_size=32), ValueError), (dict(head_dim=64), ValueError)])
def test_cache_refuses_other_formats(kw, error):
    args = dict(head_dim=128, page_size=64, dtype=torch.bfloat16) | kw
    with pytest.raises(error):
        gfa.KV4Cache(pages_of(), **args)


def test_cache_refuses_other_tensors():
    ok = dict(head_dim=128, page_size=64, dtype=torch.bfloat16)
    assert gfa.KV4Cache(pages_of(), **ok).num_pages == 4 and gfa.KV4Cache(pages_of(), **ok).num_kv_heads == 2
    for bad in (pages_of().int(), pages_of().flatten(), pages_of().transpose(0, 2), pages_of()[..., :544]):
        with pytest.raises(ValueError):
            gfa.KV4Cache(bad, **ok)
    for kw in (dict(num_pages=0), dict(num_kv_heads=0), dict(num_pages=2 ** 26)):
        with pytest.raises(ValueError):
            gfa.kv4_alloc(**(dict(num_pages=3, num_kv_heads=1, head_dim=64, device="cpu") | kw))


def test_cpu_tensors_are_refused():
    cache = gfa.KV4Cache(pages_of(), head_dim=128, page_size=64, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16)
    calls = [lambda: gfa.kv4_plan(i32(1), i32(1), i32(1, 1), i32(1), i32(2), page_size=64, max_new=1),
             lambda: gfa.kv4_append(cache, k, k, i32(1, 1)),
             lambda: gfa.kv4_read(cache, i32(1, 1), i32(1), 1),
             lambda: gfa.attention_flash_gqa_kv4(k, cache, i32(1, 1), i32(1))]
    for call in calls:
        with pytest.raises(RuntimeError, match="CPU"):
            call()
    with pytest.raises(TypeError):
        gfa.kv4_append(cache, [1.0], k, i32(1, 1))


FAKE = 0x100000  # never dereferenced: validation fails first


def _message():
    return _lib.load().gqafa_last_error().decode()


@pytest.mark.parametrize("heads,dim,page,want", [(4, 512, 64, 2 * 4 * 4 * 8 * 544), (1, 64, 16, 2 * 544),
                                                 (3, 128, 256, 2 * 3 * 16 * 2 * 544), (0, 64, 16, -1), (1, 96, 16, -1),
                                                 (1, 64, 8, -1), (1, 64, 24, -1)])
def test_page_bytes(heads, dim, page, want):
    assert _lib.load().gqafa_kv4_page_bytes(heads, dim, page) == want


@pytest.mark.parametrize("over,code,msg", [
    (dict(B=0), _lib.GQAFA_ERR_INVALID, "positive"), (dict(max_new=0), _lib.GQAFA_ERR_INVALID, "positive"),
    (dict(page=40), _lib.GQAFA_ERR_UNSUPPORTED, "page_size"), (dict(cols=0), _lib.GQAFA_ERR_INVALID, "columns"),
    (dict(B=2 ** 16, cols=2 ** 16), _lib.GQAFA_ERR_INVALID, "out of range"),
    (dict(F=0), _lib.GQAFA_ERR_INVALID, "free_pages"), (dict(F=2 ** 30), _lib.GQAFA_ERR_INVALID, "free_pages"),
    (dict(lens=None), _lib.GQAFA_ERR_INVALID, "kv_lens"), (dict(slots=FAKE + 2), _lib.GQAFA_ERR_INVALID, "slot_map"),
    (dict(stride=-1), _lib.GQAFA_ERR_INVALID, "stride")])
def test_plan_validation(over, code, msg):
    a = dict(lens=FAKE, stride=4, B=2, cols=4, F=8, page=64, max_new=3, slots=FAKE) | over
    rc = _lib.load().gqafa_kv4_plan(a["lens"], FAKE, FAKE, a["stride"], FAKE, FAKE, a["B"], a["cols"], a["F"], a["page"],
                                    a["max_new"], FAKE, FAKE, FAKE, a["slots"], FAKE, FAKE, FAKE, None)
    assert rc == code and msg in _message()


@pytest.mark.parametrize("over,code,msg", [
    (dict(D=96), _lib.GQAFA_ERR_UNSUPPORTED, "head_dim"), (dict(dtype=2), _lib.GQAFA_ERR_INVALID, "dtype"),
    (dict(N=0), _lib.GQAFA_ERR_INVALID, "positive"), (dict(Hkv=0), _lib.GQAFA_ERR_INVALID, "heads_kv"),
    (dict(pages=None), _lib.GQAFA_ERR_INVALID, "pages"), (dict(pages=FAKE + 8), _lib.GQAFA_ERR_INVALID, "aligned"),
    (dict(num_pages=0), _lib.GQAFA_ERR_INVALID, "num_pages"), (dict(num_pages=2 ** 31), _lib.GQAFA_ERR_INVALID, "num_pages"),
    (dict(k=FAKE + 4), _lib.GQAFA_ERR_INVALID, "aligned"), (dict(ks=(128, 64, 12, 1)), _lib.GQAFA_ERR_INVALID, "strides"),
    (dict(ks=(128, 64, 64, 2)), _lib.GQAFA_ERR_INVALID, "last"), (dict(ks=(0, 64, 64, 1)), _lib.GQAFA_ERR_INVALID, "strides"),
    (dict(slots=None), _lib.GQAFA_ERR_INVALID, "slot_map"), (dict(B=70000), _lib.GQAFA_ERR_INVALID, "65535")])
def test_append_validation(over, code, msg):
    a = dict(k=FAKE, ks=(1024, 512, 64, 1), slots=FAKE, pages=FAKE, num_pages=9, B=2, Hkv=2, N=8, D=64, page=64, dtype=1) | over
    st = _lib.strides_arg((1024, 512, 64, 1))
    rc = _lib.load().gqafa_kv4_append(a["k"], _lib.strides_arg(a["ks"]), FAKE, st, a["slots"], 8, a["pages"], a["num_pages"],
                                      a["B"], a["Hkv"], a["N"], a["D"], a["page"], a["dtype"], None)
    if over.get("B") == 70000:  # passes validation up to the launch shape, which needs a device first
        assert rc != _lib.GQAFA_OK
        return
    assert rc == code and msg in _message()


@pytest.mark.parametrize("over,code,msg", [
    (dict(n=0), _lib.GQAFA_ERR_INVALID, "positive"), (dict(B=2 ** 31 - 1, n=2 ** 31 - 1), _lib.GQAFA_ERR_INVALID, "range"),
    (dict(lens=None), _lib.GQAFA_ERR_INVALID, "kv_lens"),
    (dict(k=FAKE + 16), _lib.GQAFA_ERR_INVALID, "32-byte"), (dict(v=None), _lib.GQAFA_ERR_INVALID, "outputs"),
    (dict(cols=2 ** 27), _lib.GQAFA_ERR_INVALID, "columns"), (dict(starts=FAKE + 1), _lib.GQAFA_ERR_INVALID, "starts")])
def test_read_validation(over, code, msg):
    a = dict(lens=FAKE, starts=None, k=FAKE, v=FAKE, cols=4, n=8, B=2) | over
    rc = _lib.load().gqafa_kv4_read(FAKE, 9, FAKE, 4, a["cols"], a["lens"], a["starts"], a["k"], a["v"], a["B"], 2, a["n"],
                                    64, 64, 1, None)
    assert rc == code and msg in _message()


@pytest.mark.parametrize("over,code,msg", [
    (dict(Hq=5), _lib.GQAFA_ERR_INVALID, "multiple"), (dict(Hq=2 ** 31 - 2, N=2 ** 31 - 1), _lib.GQAFA_ERR_INVALID, "range"),
    (dict(N=0), _lib.GQAFA_ERR_INVALID, "positive"),
    (dict(D=32), _lib.GQAFA_ERR_UNSUPPORTED, "head_dim"), (dict(page=17), _lib.GQAFA_ERR_UNSUPPORTED, "page_size"),
    (dict(scale=0.0), _lib.GQAFA_ERR_INVALID, "softmax_scale"), (dict(scale=math.nan), _lib.GQAFA_ERR_INVALID, "softmax_scale"),
    (dict(window=-1), _lib.GQAFA_ERR_INVALID, "window"), (dict(max_len=-1), _lib.GQAFA_ERR_INVALID, "max_kv_len"),
    (dict(q=None), _lib.GQAFA_ERR_INVALID, "q: null"), (dict(o=FAKE + 2), _lib.GQAFA_ERR_INVALID, "o: data pointer"),
    (dict(lse=FAKE + 2), _lib.GQAFA_ERR_INVALID, "lse"), (dict(q_lens=FAKE + 2), _lib.GQAFA_ERR_INVALID, "q_lens")])
def test_attend_validation(over, code, msg):
    a = dict(q=FAKE, o=FAKE, lse=None, q_lens=None, Hq=4, N=3, D=64, page=64, max_len=0, scale=0.1, window=0) | over
    st = _lib.strides_arg((4 * 3 * 64, 3 * 64, 64, 1))
    rc = _lib.load().gqafa_kv4_attend(a["q"], st, FAKE, 9, FAKE, 4, 4, FAKE, a["q_lens"], a["o"], st, a["lse"], 2, a["Hq"], 2,
                                      a["N"], a["D"], a["page"], a["max_len"], a["scale"], 1, a["window"], 1, FAKE, 1 << 30, None)
    assert rc == code and msg in _message()
