"""An STU layer whose queries and keys are normed and rotated by their position, trained on jagged batches and
served from a paged 4-bit cache.

``STULayer`` with two steps between its projection and its attention (``qk_norm_rotary``) and another way to
serve: ``paged_forward`` takes any number of new rows of every user, writes their K (normed and rotated on the
way) and V into the user's pages and attends over them.  The reference's layer has neither; its cached path
(generative_recommenders/modules/stu.py:358-424) is the one of ``STULayer``.
"""

from dataclasses import dataclass
from typing import Optional

import torch

from .common import as_dtype, span
from .hstu_attention import hstu_mha
from .hstu_compute import hstu_compute_output, hstu_compute_uqvk
from .paged_cache import PagedKVCache, append_paged_kv, paged_mha
from .qk_norm_rotary import qk_norm_rotary, rotary_tables
from .stu import STULayer, STULayerConfig


@dataclass
class RotarySTULayerConfig(STULayerConfig):
    max_positions: int = 16384      # rows of the rotation's tables
    rotary_dim: Optional[int] = None  # leading values of a head that are rotated; None: all of them
    rotary_base: float = 10000.0


def _new_positions(cached_lengths: torch.Tensor, new_offsets: torch.Tensor, rows: int) -> torch.Tensor:
    """The position of every new row; of rows that no sequence has (padding) any number."""
    row = torch.arange(rows, device=new_offsets.device)
    # (-1 before the first offset and B past the last: both are the entry that is added at the end)
    seq = torch.searchsorted(new_offsets, row.to(new_offsets.dtype), right=True) - 1
    first = torch.nn.functional.pad(cached_lengths - new_offsets[:-1].to(cached_lengths.dtype), (0, 1))
    return first[seq] + row.to(cached_lengths.dtype)


class RotarySTULayer(STULayer):
    """``STULayer`` with weights for the norms of q and k (``_q_norm_weight``, ``_k_norm_weight``, one entry per
    value of a head) and rotated positions; ``attention_dim`` and ``hidden_dim`` are the same.

    The projection, the norms and the attention are separate stages: ``recompute_uvqk`` and ``recompute_normed_x``, which
    say what a fused one keeps for its backward, change nothing here, nor does ``sort_by_length``, which no kernel needs."""

    def __init__(self, config: RotarySTULayerConfig, is_inference: bool = False) -> None:
        if config.rel_bias_buckets > 0:
            raise ValueError("rotated positions and a relative bias table are alternatives")
        if config.attention_dim != config.hidden_dim:
            raise ValueError("the paged cache holds K and V of one head dimension")
        super().__init__(config, is_inference)
        self._q_norm_weight = torch.nn.Parameter(torch.ones(config.attention_dim))
        self._k_norm_weight = torch.nn.Parameter(torch.ones(config.attention_dim))
        self._rotary_base = config.rotary_base
        cos, sin = rotary_tables(config.max_positions, config.rotary_dim or config.attention_dim, config.rotary_base)
        self.register_buffer("_cos", cos, persistent=False)
        self.register_buffer("_sin", sin, persistent=False)

    def _apply(self, fn, recurse=True):
        # a change of the module's dtype is one of its parameters: the tables stay in 32 bits
        super()._apply(fn, recurse)
        if self._cos.dtype != torch.float32:
            n, dim = self._cos.shape[0], 2 * self._cos.shape[1]
            self._cos, self._sin = rotary_tables(n, dim, self._rotary_base, device=self._cos.device)
        return self

    def new_cache(self, num_pages: int, page_size: int = 64, device="cuda") -> PagedKVCache:
        return PagedKVCache.allocate(num_pages, self._num_heads, self._attention_dim, page_size, device)

    def _uqvk(self, x):
        with span("## stu_compute_uqvk ##"):
            return hstu_compute_uqvk(
                x=x, norm_weight=as_dtype(self._input_norm_weight, x.dtype),
                norm_bias=as_dtype(self._input_norm_bias, x.dtype), norm_eps=1e-6, num_heads=self._num_heads,
                attn_dim=self._attention_dim, hidden_dim=self._hidden_dim,
                uvqk_weight=as_dtype(self._uvqk_weight, x.dtype), uvqk_bias=as_dtype(self._uvqk_beta, x.dtype),
                kernel=self._hammer_kernel)

    def _head_weight(self, w, like):
        # (q and k may be of another type than the parameters, as under autocast; the kernels take fp32 or theirs)
        return w if w.dtype == like.dtype else as_dtype(w, torch.float32)

    def _output(self, attn, u, x):
        with span("## stu_compute_output ##"):
            return hstu_compute_output(
                attn=attn.reshape(-1, self._hidden_dim * self._num_heads), u=u, x=x,
                norm_weight=as_dtype(self._output_norm_weight, x.dtype),
                norm_bias=as_dtype(self._output_norm_bias, x.dtype), norm_eps=1e-6,
                output_weight=as_dtype(self._output_weight, x.dtype), num_heads=self._num_heads,
                linear_dim=self._hidden_dim, dropout_ratio=self._output_dropout_ratio, training=self.training,
                concat_u=True, concat_x=True, mul_u_activation_type="none", group_norm=self._use_group_norm,
                recompute_y_in_backward=self._recompute_y, kernel=self._hammer_kernel)

    def forward(self, x, x_lengths, x_offsets, max_seq_len, num_targets, max_kv_caching_len=0, kv_caching_lengths=None):
        """``STULayer.forward``; row i of a sequence is at position i.  The 16-bit cache is not kept."""
        if kv_caching_lengths is not None:
            raise NotImplementedError("RotarySTULayer serves from a paged cache: paged_forward")
        u, q, k, v = self._uqvk(x)
        rows = torch.arange(x.shape[0], device=x.device)
        offsets = x_offsets.to(rows.dtype)
        positions = rows - offsets[torch.searchsorted(offsets, rows, right=True) - 1]
        with span("## qk_norm_rotary ##"):
            q, k = qk_norm_rotary(q.view(-1, self._num_heads, self._attention_dim),
                                  k.view(-1, self._num_heads, self._attention_dim), positions, self._cos, self._sin,
                                  self._head_weight(self._q_norm_weight, q), self._head_weight(self._k_norm_weight, k),
                                  kernel=self._hammer_kernel)
        with span("## hstu_mha ##"):
            attn = hstu_mha(max_seq_len=max_seq_len, alpha=self._attn_alpha, q=q, k=k,
                            v=v.view(-1, self._num_heads, self._hidden_dim), seq_offsets=x_offsets, causal=self._causal,
                            training=self.training, num_targets=num_targets if self._target_aware else None,
                            max_attn_len=self._max_attn_len, contextual_seq_len=self._contextual_seq_len,
                            kernel=self._hammer_kernel)
        return self._output(attn, u, x)

    def cached_forward(self, delta_x, num_targets, max_kv_caching_len=0, kv_caching_lengths=None):
        raise NotImplementedError("RotarySTULayer serves from a paged cache: paged_forward")

    @torch.no_grad()
    def paged_forward(
        self,
        new_x: torch.Tensor,
        cache: PagedKVCache,
        page_table: torch.Tensor,
        cached_lengths: torch.Tensor,
        new_offsets: torch.Tensor,
        max_seq_len: int,
        num_targets: Optional[torch.Tensor] = None,
    ) -> torch.Tensor:
        """The layer on the rows ``new_offsets[b] .. new_offsets[b + 1]`` of ``new_x``, which follow the
        ``cached_lengths[b]`` rows of sequence b that the cache holds; theirs are in it afterwards.

        ``page_table`` names pages for all of them.  ``max_seq_len`` is what divides SiLU's weights, the one that
        the layer was trained with.  Candidates (``num_targets``) that are not to stay are overwritten by the next
        call when it is given the same ``cached_lengths``.  Rows past ``new_offsets[-1]`` (padding) are in no sequence:
        nothing is cached for them and their attention is zeros."""
        torch._assert(self._causal, "only support causal attention")
        H, d = self._num_heads, self._attention_dim
        u, q, k, v = self._uqvk(new_x)
        lengths = cached_lengths + (new_offsets[1:] - new_offsets[:-1]).to(cached_lengths.dtype)
        positions = _new_positions(cached_lengths, new_offsets, new_x.shape[0])
        with span("## qk_norm_rotary ##"):
            q, _ = qk_norm_rotary(q.view(-1, H, d), None, positions, self._cos, self._sin,
                                  self._head_weight(self._q_norm_weight, q), kernel=self._hammer_kernel)
        with span("## append_paged_kv ##"):
            append_paged_kv(cache, k.view(-1, H, d), v.view(-1, H, d), page_table, cached_lengths, new_offsets, self._cos,
                            self._sin, k_weight=self._head_weight(self._k_norm_weight, k), kernel=self._hammer_kernel)
        with span("## paged_mha ##"):
            attn = paged_mha(max_seq_len, self._attn_alpha, q, cache, page_table, lengths, new_offsets,
                             num_targets if self._target_aware else None, self._max_attn_len, self._contextual_seq_len,
                             kernel=self._hammer_kernel)
        return self._output(attn, u, new_x)
