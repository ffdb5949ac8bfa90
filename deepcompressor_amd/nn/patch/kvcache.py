"""Keys and values of past tokens held in 8 bits, and the attention over them.  ``ScaleDotProductAttention`` is where the
calibration quantizes keys and values; this is the cache that a decoder keeps of them (no counterpart in the
reference, which leaves the cache to the serving back end)."""

from __future__ import annotations

import torch

from ...engine_fp8 import E4M3, F32, kv_append, kv_attention

__all__ = ["Fp8KVCache"]


class Fp8KVCache:
    """Pages of ``page_size`` (16, 32, 64 or 128) tokens as e4m3 codes, with a power-of-two scale for each page and head.

    ``k_codes`` float8_e4m3fn [page][head][token][channel], ``v_codes`` [page][head][channel][token] (transposed),
    ``k_scales`` / ``v_scales`` float32 [page][head].  Which pages a sequence has is the caller's: ``block_table`` int32
    [sequence][column] lists them in the tokens' order; an entry outside the pool (-1) is no page, its tokens are neither
    written nor seen.  Everything is read on the device: the calls do not wait for it and can be captured in a graph.

    Tokens are [sequence][token][head][channel], the same number for each sequence, or packed [token][head][channel] with
    ``starts`` int32 [sequences + 1]: sequence i has tokens starts[i] .. starts[i + 1] - 1."""

    def __init__(self, num_pages: int, num_heads: int, head_dim: int, page_size: int = 64,
                 device: torch.device | str = "cuda") -> None:
        make = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device=device).view(E4M3)  # noqa: E731
        self._set(make(num_pages, num_heads, page_size, head_dim), torch.ones((num_pages, num_heads), device=device),
                  make(num_pages, num_heads, head_dim, page_size), torch.ones((num_pages, num_heads), device=device))

    @staticmethod
    def from_buffers(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor) -> "Fp8KVCache":
        """A cache over tensors that the caller keeps (they are used, not copied).  Scales are positive and
        normal (appends make powers of two)."""
        cache = Fp8KVCache.__new__(Fp8KVCache)
        cache._set(k_codes, k_scales, v_codes, v_scales)
        return cache

    def _set(self, k_codes, k_scales, v_codes, v_scales) -> None:
        shape = k_codes.shape
        if len(shape) != 4:
            raise ValueError("k_codes are [page][head][token][channel]")
        pool, heads, page, dim = shape
        if pool < 1 or heads < 1:
            raise ValueError("a cache has at least one page and one head")
        if page not in (16, 32, 64, 128):
            raise ValueError(f"pages hold 16, 32, 64 or 128 tokens, not {page}")
        if dim not in (64, 128):
            raise ValueError(f"heads have 64 or 128 channels, not {dim}")
        per_head = (pool, heads)
        if (k_codes.dtype != E4M3 or v_codes.dtype != E4M3 or k_scales.dtype != F32 or v_scales.dtype != F32
                or v_codes.shape != (pool, heads, dim, page) or k_scales.shape != per_head or v_scales.shape != per_head):
            raise ValueError(f"expected float8_e4m3fn codes {(pool, heads, page, dim)} and {(pool, heads, dim, page)} (values transposed) "
                             f"and float32 scales {(pool, heads)}; got {k_codes.dtype}, {v_codes.dtype} of {tuple(v_codes.shape)}, "
                             f"{k_scales.dtype} of {tuple(k_scales.shape)}, {v_scales.dtype} of {tuple(v_scales.shape)}")
        at = k_codes.get_device()
        if (v_codes.get_device() != at or k_scales.get_device() != at or v_scales.get_device() != at or not k_codes.is_contiguous()
                or not v_codes.is_contiguous() or not k_scales.is_contiguous() or not v_scales.is_contiguous()):
            raise ValueError("a cache's tensors are contiguous and on one device")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    def append(self, key: torch.Tensor, value: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
               starts: torch.Tensor | None = None) -> None:
        """Write each sequence's new tokens behind its ``lengths`` older ones (int32 [sequences]).  A page's scale is the
        smallest power of two that takes its values to 448 or less: its first token sets it, a later, larger one raises
        it and the page's codes are rescaled.  Tokens behind the table's last column are dropped.  A value that is not
        finite is stored as NaN.  A page may be written by one sequence only (one that is shared, for a common
        beginning, must be full)."""
        kv_append(key, value, self.k_codes, self.k_scales, self.v_codes, self.v_scales, block_table, lengths, starts)

    def attend(self, query: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *, starts: torch.Tensor | None = None,
               scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale * q k') v for the queries of each sequence's last tokens, ``lengths`` counting all of its tokens in
        the cache, those of the queries included (of more than the table holds, those that it holds are seen).  ``causal``: query j of n
        sees the tokens before lengths - n + j + 1.
        Query head h reads cache head h // (query heads // cache heads).  A query that sees no token gives 0.
        ``scale``: head_dim ** -0.5 by default.  ``out``: written in place, rows of a packed tensor that no sequence has are
        left as they were (without ``out`` they are 0); it may be ``query`` itself, and shares no memory with it, or with the
        cache, otherwise.  Probabilities are rounded to the query's type, their sums are float32.  Work on a batch of chunks begins with its last sequence: the longest are best
        listed last."""
        scale = self.k_codes.shape[3] ** -0.5 if scale is None else scale
        return kv_attention(query, self.k_codes, self.k_scales, self.v_codes, self.v_scales, block_table, lengths, starts,
                            scale, causal, out)
