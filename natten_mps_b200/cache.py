"""A paged key/value cache for ``na1d_append`` and ``na1d_paged``: the pools on the GPU, the pages' bookkeeping on the host."""
from __future__ import annotations

from typing import List, NamedTuple, Sequence, Union

import torch


class CacheLayer(NamedTuple):
    """One layer's pools with the page table and lengths that all layers share, as the operators take them."""
    key_cache: torch.Tensor
    value_cache: torch.Tensor
    page_table: torch.Tensor
    cache_lens: torch.Tensor
    seq_lens: torch.Tensor


class PagedCache:
    """Keys and values of ``batch`` sequences of up to ``max_length`` tokens in ``num_pages`` pages of ``page_size``
    tokens, for ``layers`` layers (which share the page table: a page holds the same tokens in each).

    ``extend(new)`` makes room for the next tokens, before the layers run; ``layer(i)`` is what a layer's operators take::

        cache.extend([len(p) for p in prompts])            # or one number for all
        for i, block in enumerate(blocks):
            x = block(x, cache=cache.layer(i))             # na1d_append, then na1d_paged

    ``page_table [batch, n]``, ``cache_lens [batch]`` and ``seq_lens [batch]`` are int32 tensors on the device that are
    updated in place on the current stream, so that a captured step can be replayed after the next ``extend``.  Pages that
    are not there are -1 in the table."""

    def __init__(self, batch: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, max_length: int, *,
                 layers: int = 1, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        for name, value in (("batch", batch), ("num_pages", num_pages), ("page_size", page_size), ("num_kv_heads", num_kv_heads),
                            ("head_dim", head_dim), ("max_length", max_length), ("layers", layers)):
            if isinstance(value, bool) or not isinstance(value, int) or value < 1:
                raise ValueError(f"{name} must be a positive integer, got {value}.")
        self.batch, self.num_pages, self.page_size, self.max_length = batch, num_pages, page_size, max_length
        # zeros, not empty: what no token was written to is never attended to, but it should not hold another tensor's data
        self.pools = torch.zeros(layers, 2, num_pages, page_size, num_kv_heads, head_dim, dtype=dtype, device=device)
        self._width = -(-max_length // page_size)
        self.page_table = torch.full((batch, self._width), -1, dtype=torch.int32, device=device)
        self.cache_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[-1] * self._width for _ in range(batch)]
        self._lens: List[int] = [0] * batch
        self._trimmed: List[int] = [0] * batch               # pages of each sequence given back from its front

    def __len__(self) -> int:
        return self.batch

    @property
    def lengths(self) -> List[int]:
        """Tokens of each sequence (host copy)."""
        return list(self._lens)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, index: int = 0) -> CacheLayer:
        pool = self.pools[index]
        return CacheLayer(pool[0], pool[1], self.page_table, self.cache_lens, self.seq_lens)

    def extend(self, new: Union[int, Sequence[int]]) -> None:
        """Room for ``new`` further tokens a sequence (one number, or one for each; 0 leaves a sequence alone).  Raises
        ``ValueError`` past ``max_length`` and ``RuntimeError`` without enough free pages, and then changes nothing."""
        counts = [new] * self.batch if isinstance(new, int) else [int(n) for n in new]
        if len(counts) != self.batch or any(n < 0 for n in counts):
            raise ValueError(f"new must be a non-negative count, or one for each of the {self.batch} sequences.")
        for b, n in enumerate(counts):
            if self._lens[b] + n > self.max_length:
                raise ValueError(f"sequence {b} would have {self._lens[b] + n} tokens, max_length is {self.max_length}.")
        wanted = [range(-(-self._lens[b] // self.page_size), -(-(self._lens[b] + n) // self.page_size)) for b, n in enumerate(counts)]
        if sum(len(w) for w in wanted) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(len(w) for w in wanted)} are needed.")
        for b, n in enumerate(counts):
            for slot in wanted[b]:
                self._pages[b][slot] = self._free.pop()
            self._lens[b] += n
        if any(len(w) for w in wanted):
            self._upload_table()
        self._upload(self.cache_lens, self._lens)
        self._upload(self.seq_lens, counts)

    def reset(self, sequence: int) -> None:
        """Forget a sequence and give its pages back."""
        self._give_back(sequence, self._width)
        self._lens[sequence] = 0
        self._trimmed[sequence] = 0
        self._upload_table()
        self._upload(self.cache_lens, self._lens)
        counts = self.seq_lens.clone()
        counts[sequence] = 0
        self.seq_lens.copy_(counts)

    def trim(self, keep: int) -> None:
        """Give back the pages that lie wholly in front of each sequence's last ``keep`` tokens: behind a sliding window of
        ``kernel_size`` and ``dilation`` the next token still needs ``(kernel_size - 1) * dilation`` of them."""
        if keep < 0:
            raise ValueError("keep must not be negative.")
        for b in range(self.batch):
            self._give_back(b, max(0, self._lens[b] - keep) // self.page_size)
        self._upload_table()

    def _give_back(self, sequence: int, pages: int) -> None:
        for slot in range(self._trimmed[sequence], pages):
            page = self._pages[sequence][slot]
            if page >= 0:
                self._free.append(page)
                self._pages[sequence][slot] = -1
        self._trimmed[sequence] = max(self._trimmed[sequence], pages)

    def _upload_table(self) -> None:
        self._upload(self.page_table, self._pages)

    @staticmethod
    def _upload(target: torch.Tensor, values) -> None:
        target.copy_(torch.tensor(values, dtype=torch.int32))


__all__ = ["CacheLayer", "PagedCache"]
