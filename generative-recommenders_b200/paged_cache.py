"""K and V of served sequences in pages of 4-bit codes, and the attention that reads them.

The reference's cached inference keeps one jagged 16-bit K and V per layer and copies both when rows join them
(generative_recommenders/modules/stu.py:84-173).  Here a user's rows lie in pages of a common pool, appending
writes the new rows alone, and a cached row takes ``d + 4 d / 64`` bytes a head instead of ``4 d``.

A page holds ``page_size`` consecutive positions of one sequence.  K and V are rounded in groups of 64 values to
``(code - 8) * scale`` with codes 1 .. 15 and a bfloat16 scale, max |x| / 7 of the group.  ``page_table[b]`` names
the pages of sequence b in order; which pages are free is the caller's business.
"""

from typing import Optional, Tuple

import torch

from . import _cabi
from . import hstu_attention as _attention
from .common import HammerKernel, _require_cuda_backend

_GROUP = 64
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)


class PagedKVCache:
    """A pool of pages: ``pages`` is uint8 ``[num_pages, heads, page_bytes(page_size, head_dim)]``, contiguous."""

    __slots__ = ("pages", "page_size", "head_dim")

    def __init__(self, pages: torch.Tensor, page_size: int, head_dim: int) -> None:
        if page_size not in PAGE_SIZES:
            raise ValueError("a page has one of %s positions, not %r" % (PAGE_SIZES, page_size))
        if head_dim not in HEAD_DIMS:
            raise ValueError("a head has one of %s values, not %r" % (HEAD_DIMS, head_dim))
        _cabi.host().check_pages(pages, page_size, head_dim)
        self.pages, self.page_size, self.head_dim = pages, page_size, head_dim

    @staticmethod
    def page_bytes(page_size: int, head_dim: int) -> int:
        """Bytes of one head's K and V in a page: codes, then scales."""
        return 2 * page_size * (head_dim // 2 + 2 * (head_dim // _GROUP))

    @classmethod
    def allocate(cls, num_pages: int, num_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> "PagedKVCache":
        """A pool with undefined contents (nothing reads a position that was not appended)."""
        return cls(torch.empty((num_pages, num_heads, cls.page_bytes(page_size, head_dim)), dtype=torch.uint8, device=device),
                   page_size, head_dim)

    @property
    def num_pages(self) -> int:
        return self.pages.shape[0]

    @property
    def num_heads(self) -> int:
        return self.pages.shape[1]


def append_paged_kv(
    cache: PagedKVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    cached_lengths: torch.Tensor,
    new_offsets: torch.Tensor,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    kernel: HammerKernel = HammerKernel.CUDA,
) -> None:
    """Rows ``new_offsets[b] .. new_offsets[b + 1]`` of ``k``, ``v [rows, heads, d]`` become positions
    ``cached_lengths[b] ..`` of sequence b, K normed (``k_weight``) and rotated (``cos``, ``sin``) by its position
    first, as :func:`qk_norm_rotary` does it, both optional.

    ``page_table`` is int32 ``[B, pages]``; lengths and offsets are int32 or int64.  A row whose position has no
    page of the pool is not written.  A group with an infinity or a NaN stands for NaN afterwards, one too small
    for a scale for zeros.  Rows of one call must not share a position."""
    _require_cuda_backend(kernel)
    _cabi.host().paged_append(cache.pages, cache.page_size, cache.head_dim, k, v, page_table, cached_lengths, new_offsets,
                              cos, sin, bool(interleaved), k_weight, float(eps))


def read_paged_kv(
    cache: PagedKVCache,
    page_table: torch.Tensor,
    seq_offsets: torch.Tensor,
    total_rows: int,
    dtype: torch.dtype = torch.bfloat16,
    kernel: HammerKernel = HammerKernel.CUDA,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of the first ``seq_offsets[b + 1] - seq_offsets[b]`` positions of every sequence: jagged
    ``k, v [total_rows, heads, d]``, as :func:`delta_hstu_mha` and ``STULayer``'s 16-bit cache have them.  Rows
    without a page of the pool are NaN, rows beyond ``seq_offsets[-1]`` zeros."""
    _require_cuda_backend(kernel)
    return _cabi.host().paged_read(cache.pages, cache.page_size, cache.head_dim, page_table, seq_offsets, int(total_rows),
                                   dtype)


def paged_mha(
    max_seq_len: int,
    alpha: float,
    q: torch.Tensor,
    cache: PagedKVCache,
    page_table: torch.Tensor,
    seq_lengths: torch.Tensor,
    q_offsets: torch.Tensor,
    num_targets: Optional[torch.Tensor] = None,
    max_attn_len: int = 0,
    contextual_seq_len: int = 0,
    activation: str = "silu",
    attn_scale: Optional[float] = None,
    kernel: HammerKernel = HammerKernel.CUDA,
) -> torch.Tensor:
    """Attention of the last rows of every sequence over the paged cache, which holds them already
    (:func:`append_paged_kv`): ``delta_hstu_mha`` with the mask, but sequences may have any number of new rows.

    Rows ``q_offsets[b] .. q_offsets[b + 1]`` of ``q [rows, H, d]`` are the last positions of sequence b, which is
    ``seq_lengths[b]`` long.  ``H`` is a multiple of the cache's heads; query head h reads head
    ``h // (H / heads)``.  ``activation`` is ``"silu"``, HSTU's weights ``SiLU(alpha q.k) * attn_scale`` with
    ``attn_scale = 1 / max_seq_len`` unless given, or ``"softmax"`` of ``alpha q.k`` over what the row sees.
    The last ``num_targets[b]`` positions see none of each other, ``max_attn_len > 0`` limits how far back a row
    sees and ``contextual_seq_len`` is the length of the contextual prefix.

    A row that sees nothing gives zeros, one that sees a position without a page of the pool NaN; table entries
    that no row sees (those that a window has left behind) may hold anything.  The same call gives the same bits;
    where a long sequence's sums are cut depends on the work of the whole batch, so in another batch a row may differ
    in the last of them.  A group of V that is NaN makes that group's columns NaN of the rows that see it.  Rows of q before
    the first offset and past the last are zeros.

    Scores and sums are fp32.  Weights are rounded to 16 bits (float32 q: 24); from 17 rows a sequence of the batch on, with
    16-bit q and heads of 64 or 128, to 11 bits, with SiLU's tanh off by 2^-11 of half the score as in
    :func:`hstu_mha`'s 16-bit kernels.  Scales of any size are exact there down to 2^-22 of the largest of 128
    positions' (smaller ones lose a bit for each power of two).  No gradient: this is the inference path."""
    _require_cuda_backend(kernel)
    torch._assert(max_seq_len > 0, "max_seq_len must be larger than 0")
    torch._assert(max_attn_len >= 0 and contextual_seq_len >= 0, "max_attn_len and contextual_seq_len must not be negative")
    if activation not in ("silu", "softmax"):
        raise ValueError("activation must be 'silu' or 'softmax', not %r" % (activation,))
    return _cabi.host().paged_attention(
        q.detach(), cache.pages, cache.page_size, cache.head_dim, page_table, seq_lengths, q_offsets, num_targets,
        float(alpha), 1.0 / max_seq_len if attn_scale is None else float(attn_scale), int(max_attn_len),
        int(contextual_seq_len), activation == "softmax", _attention._CHECK_STATUS)
