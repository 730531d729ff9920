"""Serving from a paged KV cache held in 4 bits, on B200 (sm_100a).

The reference has no cache of its own (attention.py:552-553 reads the key
length off the queries); ``attention_flash_gqa`` here takes a dense 16-bit one.
This module adds a paged cache at 4.25 bits a value and what a serving loop
runs on it:

    cache = kv4_alloc(num_pages, num_kv_heads, head_dim, page_size)
    plan = kv4_plan(kv_lens, new_lens, block_table, free_pages, free_state,
                    page_size=cache.page_size, max_new=n)
    kv4_append(cache, k, v, plan.slot_map)                     # once per layer
    o = attention_flash_gqa_kv4(q, cache, plan.block_table, plan.kv_lens,
                                causal=True, q_lens=plan.new_lens)

Shapes follow ``attention_flash_gqa``: q (B, H_Q, N, D), k and v
(B, H_KV, N, D), fp16 or bf16, D in {64, 128, 256, 512}; a batch whose
requests bring different numbers of tokens is padded to N, with the slots of
the padding -1 and the true counts in ``q_lens``. Lengths, tables and slots
are int32 CUDA tensors and stay on the GPU: no call synchronises, so a whole
step can be captured into a CUDA graph.

Number format: groups of 64 values along head_dim are held as ``s * (c - z)``
with 4-bit codes c, a zero point z in 0..15 and a scale s of 4 significant bits
(csrc/kv4_layout.cuh). Those values are exact in fp16 and bf16: what
``kv4_read`` returns is bit for bit what the attention uses.

Everything runs through ``torch.ops.gqafa.kv4_*`` over the C ABI
(include/gqa_fa_b200.h); there is no backward and no CPU path.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from .attention import _DTYPES

__all__ = ["KV4Cache", "KV4Plan", "kv4_alloc", "kv4_plan", "kv4_append", "kv4_read", "attention_flash_gqa_kv4"]

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256, 512)
BLOCK_TOKENS = 16
GROUP_BYTES = 544  # a block's bytes per 64 dims: 16 tokens x 64 codes, 16 scale words


class KV4Cache:
    """Pages of one layer: ``pages`` is a contiguous uint8 CUDA tensor
    (num_pages, 2 (keys, values), H_KV, page_size / 16, head_dim / 64 * 544).

    Slots that were never written hold whatever the memory held; the kernels
    never use them beyond the requests' lengths."""

    __slots__ = ("pages", "head_dim", "page_size", "dtype")

    def __init__(self, pages: torch.Tensor, head_dim: int, page_size: int, dtype: torch.dtype):
        _check_format(head_dim, page_size, dtype)
        want = (2, page_size // BLOCK_TOKENS, head_dim // 64 * GROUP_BYTES)
        if pages.dtype != torch.uint8 or pages.dim() != 5:
            raise ValueError(f"pages must be a 5-D uint8 tensor, got {pages.dtype} {tuple(pages.shape)}")
        if (pages.shape[1], pages.shape[3], pages.shape[4]) != want or not pages.is_contiguous():
            raise ValueError(
                f"pages of head_dim {head_dim} and page_size {page_size} must be contiguous with shape "
                f"(num_pages, 2, H_KV, {want[1]}, {want[2]}), got {tuple(pages.shape)}"
            )
        if pages.data_ptr() % 16 != 0:
            raise ValueError("pages must be 16-byte aligned")
        self.pages, self.head_dim, self.page_size, self.dtype = pages, int(head_dim), int(page_size), dtype

    @property
    def num_pages(self) -> int:
        return self.pages.shape[0]

    @property
    def num_kv_heads(self) -> int:
        return self.pages.shape[2]


class KV4Plan(NamedTuple):
    """What a step needs to know about its requests (all int32 CUDA tensors)."""

    block_table: torch.Tensor  # (B, columns) pages of each request, -1 where unused
    kv_lens: torch.Tensor      # (B,) cached tokens after the step
    new_lens: torch.Tensor     # (B,) tokens the step adds (0 where refused or finished)
    slot_map: torch.Tensor     # (B, max_new) slot of each new token, -1 behind the last
    positions: torch.Tensor    # (B, max_new) position of each new token, -1 behind the last
    free_state: torch.Tensor   # (2,) start and length of the free ring after the step
    accepted: torch.Tensor     # (B,) 1, or 0 where the request was refused


def _check_format(head_dim, page_size, dtype):
    if dtype not in _DTYPES:
        raise NotImplementedError(f"dtype {dtype} is not supported (fp16, bf16)")
    if head_dim not in HEAD_DIMS:
        raise NotImplementedError(f"head_dim {head_dim} is not implemented on sm_100a (supported: 64, 128, 256, 512)")
    if page_size not in PAGE_SIZES:
        raise NotImplementedError(f"page_size {page_size} is not implemented (supported: {PAGE_SIZES})")


def _all_cuda(*tensors):
    try:
        return all([t.is_cuda for t in tensors if t is not None])
    except AttributeError:
        return False


def _refuse(**tensors):
    """Name the argument that is not a CUDA tensor."""
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise RuntimeError(
                f"{name} is on {t.device}: gemma_triton_flash_attn runs only on CUDA (sm_100a); "
                "there is no CPU fallback"
            )


def kv4_alloc(num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> KV4Cache:
    """A cache of `num_pages` pages of `page_size` tokens for one layer."""
    _check_format(head_dim, page_size, dtype)
    if num_pages <= 0 or num_kv_heads <= 0:
        raise ValueError(f"sizes must be positive (num_pages={num_pages} num_kv_heads={num_kv_heads})")
    if num_pages * page_size >= 2 ** 31:
        raise ValueError(f"num_pages * page_size must be below 2^31, got {num_pages * page_size}")
    shape = (num_pages, 2, num_kv_heads, page_size // BLOCK_TOKENS, head_dim // 64 * GROUP_BYTES)
    return KV4Cache(torch.empty(shape, dtype=torch.uint8, device=device), head_dim, page_size, dtype)


def kv4_plan(kv_lens, new_lens, block_table, free_pages, free_state, page_size: int, max_new: int) -> KV4Plan:
    """Block table, slots and positions of the next step, built on the GPU.

    kv_lens (B,): cached tokens of each request. new_lens (B,): tokens it adds
    (0..max_new), or a negative number when it is finished and gives its pages
    back. block_table (B, columns): its pages so far. free_pages: a ring of page
    ids (each below its length), free_state = (start, count) its live part.

    Requests take free pages in request order. A request is refused (accepted
    0, nothing added) when its length would pass the table or max_new, or when
    the pages wanted by it and those before it pass the free count; pages given
    back in this step are free from the next one on. The inputs stay as they
    are, but for the ring's dead part, where returned pages are written: the
    next step passes the same ring and the returned ``free_state``.
    """
    if not _all_cuda(kv_lens, new_lens, block_table, free_pages, free_state):
        _refuse(kv_lens=kv_lens, new_lens=new_lens, block_table=block_table, free_pages=free_pages,
                free_state=free_state)
    if page_size not in PAGE_SIZES:
        raise NotImplementedError(f"page_size {page_size} is not implemented (supported: {PAGE_SIZES})")
    return KV4Plan._make(
        _lib.ops().kv4_plan(kv_lens, new_lens, block_table, free_pages, free_state, page_size, max_new))


def kv4_append(cache: KV4Cache, k, v, slot_map) -> None:
    """Quantise new keys and values (B, H_KV, N, D) into the cache.

    slot_map (B, N): the slot of each token, -1 to skip it. Slots must be
    distinct (those of a plan are). A group of 64 values that holds an infinity
    or a NaN reads back as NaN."""
    if not _all_cuda(k, v, slot_map):
        _refuse(k=k, v=v, slot_map=slot_map)
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise TypeError(f"k and v must have the cache's dtype {cache.dtype}, got {k.dtype}, {v.dtype}")
    _lib.ops().kv4_append(cache.pages, k, v, slot_map, cache.page_size)


def kv4_read(cache: KV4Cache, block_table, kv_lens, max_len: int, starts=None):
    """Cached keys and values as dense (B, H_KV, max_len, D) tensors.

    Row i of request b is position starts[b] + i (starts None or negative: 0), zeros from
    kv_lens[b] on. The values are exactly those that the attention uses, so a
    prompt that attends to them through ``attention_flash_gqa`` sees what its
    later decode steps will see."""
    if not _all_cuda(block_table, kv_lens, starts):
        _refuse(block_table=block_table, kv_lens=kv_lens, starts=starts)
    return _lib.ops().kv4_read(cache.pages, block_table, kv_lens, max_len, starts, cache.page_size, cache.dtype)


def attention_flash_gqa_kv4(q, cache: KV4Cache, block_table, kv_lens, causal=False, slide_size=0, q_lens=None,
                            softmax_scale=None, return_lse=False, max_kv_len: Optional[int] = None):
    """Inference attention over the paged 4-bit cache (no autograd).

    q (B, H_Q, N, D); kv_lens (B,): cached tokens, the new ones among them.
    The first q_lens[b] rows of request b (None: all N) are its last positions:
    row r sits at kv_lens[b] - q_lens[b] + r. With ``causal`` a row sees the keys
    up to its own position, with ``slide_size > 0`` the last slide_size of
    them; without ``causal`` every row sees all keys. Rows from q_lens[b] on,
    and rows that see no key, are zeros. Rows that see a key with a group that is
    not finite are NaN, and so is their LSE; a value group that is not finite makes
    its 64 dims NaN in the rows that see its token.

    Scores, softmax and sums are held in 32 bits. Few rows: the query enters the
    scores to 2^-16 of its row's largest value (2^-24 where that is more than 32
    times the mean), and weight times scale the sums in 16 bits; many rows: the
    weights in 16 bits. Keys or values beyond 2^96 may overflow the sums.

    Returns O shaped and typed like q (and, with return_lse, the fp32 natural-log
    LSE (B, H_Q, N), -inf where no key is seen). max_kv_len: an upper bound of
    kv_lens known to the host, which sizes the launch and the workspace (default:
    the block table's capacity). It has to hold: the rows of a longer request
    may be wrong, and ``device_status`` then returns 18."""
    if not _all_cuda(q, block_table, kv_lens, q_lens):
        _refuse(q=q, block_table=block_table, kv_lens=kv_lens, q_lens=q_lens)
    if q.dim() != 4:
        raise ValueError(f"q must be 4-D (B, H, N, D), got shape {tuple(q.shape)}")
    if q.dtype != cache.dtype:
        raise TypeError(f"q must have the cache's dtype {cache.dtype}, got {q.dtype}")
    if torch.is_grad_enabled() and q.requires_grad:
        raise NotImplementedError("attention_flash_gqa_kv4 has no backward; call it under torch.no_grad()")
    window = int(slide_size) if (slide_size and causal) else 0
    if window < 0:
        raise ValueError("slide_size must be >= 0")
    if max_kv_len is not None and max_kv_len <= 0:
        raise ValueError("max_kv_len must be positive")
    scale = (1.0 / math.sqrt(q.shape[3])) if softmax_scale is None else float(softmax_scale)
    o, lse = _lib.ops().kv4_attend(q, cache.pages, block_table, kv_lens, q_lens, cache.page_size, max_kv_len or 0,
                                   bool(causal), window, scale, bool(return_lse))
    return (o, lse) if return_lse else o
