"""The attention half of a decoder layer on the HIP library: the part that the reference's layers call
the installed model for (``lyr.self_attn``, backends.py:173-196), over a paged key-value cache.

* ``rope_tables``   the angles' tables of ``_lib.head_norm_rope`` and ``_lib.append_kv``
* ``PagedKVCache``  pages of keys and values for many sequences and layers
* ``Attention``     projections, the heads' norms with the position rotation and attention: of
  packed sequences (with gradients), of prompts on their way into a cache and of one new token
  per sequence
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib, training


def rope_tables(positions: int, columns: int, theta: float = 10000.0, device: torch.device | str | None = None,
                frequencies: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) float32 [positions, columns / 2] of position x frequency, ``frequencies`` (a vector of
    columns / 2; zero: the pair stays as it is) theta^(-2 i / columns) if None.  The angles are taken in
    64 bits: in 32, one near 100,000 is off by 0.004.  ``device`` is the frequencies' if None."""
    if columns % 2 or columns < 0:
        raise ValueError(f"columns must be even, got {columns}")
    if frequencies is None:
        frequencies = theta ** (-torch.arange(0, columns, 2, dtype=torch.float64, device=device) / max(columns, 1))
    elif frequencies.shape != (columns // 2,):
        raise ValueError(f"frequencies must be [{columns // 2}], got {list(frequencies.shape)}")
    elif device is None:
        device = frequencies.device
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * frequencies.to(device, torch.float64)
    return angle.cos().float(), angle.sin().float()


class PagedKVCache:
    """Keys and values of up to ``sequences`` sequences in pages that they take as they grow.

    ``k[layer]``, ``v[layer]``: [pages, heads, page size, head size], all layers with the same page
    numbers.  ``block_table`` [sequences, pages of the longest] and ``lengths`` [sequences] (int32, on
    the device) are what ``_lib.decode_attention`` reads, in place for the cache's whole life (a captured
    graph may hold them).  The host keeps the lengths too and decides on pages, and copies what changed to
    the device on the current stream."""

    def __init__(self, layers: int, heads: int, head_size: int, pages: int, sequences: int, longest: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str | None = None) -> None:
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if min(layers, heads, head_size, pages, sequences, longest) < 1:
            raise ValueError("every size of the cache must be at least one")
        shape = (layers, pages, heads, page_size, head_size)
        self.page_size, self.longest = page_size, longest
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        width = -(-longest // page_size)
        self.block_table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._pages: list[list[int]] = [[] for _ in range(sequences)]
        self._lengths = [0] * sequences

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        self._check(sequence)
        return self._lengths[sequence]

    def append(self, counts: dict[int, int]) -> tuple[torch.Tensor, torch.Tensor]:
        """Room for counts[s] new tokens of each sequence s -> (positions, slots), int32 on the device, of
        all new tokens, sequence after sequence in the order of ``counts``.  Raises, and takes nothing,
        where the pages or the table do not suffice or a copy to the device fails."""
        size, left = self.page_size, len(self._free)
        self._check(*counts)
        for s, n in counts.items():
            if n < 0 or self._lengths[s] + n > self.longest:
                raise ValueError(f"sequence {s} has {self._lengths[s]} tokens of {self.longest}: no room for {n}")
        grown: dict[int, list[int]] = {}
        positions = [torch.empty(0, dtype=torch.int64)]
        slots = [torch.empty(0, dtype=torch.int64)]
        for s, n in counts.items():
            at, pages = self._lengths[s], self._pages[s]
            more = -(-(at + n) // size) - len(pages)
            if more > 0:
                left -= more
                if left < 0:
                    continue
                pages = grown[s] = pages + self._free[left:left + more][::-1]
            new = torch.arange(at, at + n)
            positions.append(new)
            slots.append(torch.tensor(pages, dtype=torch.int64)[new // size] * size + new % size)
        if left < 0:
            raise RuntimeError(f"{len(self._free) - left} pages are needed, {len(self._free)} are free")
        both = torch.stack((torch.cat(positions), torch.cat(slots))).to(self.lengths.device, torch.int32)
        lengths = {s: self._lengths[s] + n for s, n in counts.items()}
        self._copy(lengths, grown)
        self._keep(lengths, grown)
        del self._free[left:]
        return both[0], both[1]

    def take_back(self, counts: dict[int, int]) -> None:
        """The last counts[s] tokens of each sequence s off again, and the pages that held nothing else free:
        what undoes an ``append`` whose keys and values were not written."""
        self._check(*counts)
        for s, n in counts.items():
            if not 0 <= n <= self._lengths[s]:
                raise ValueError(f"sequence {s} has {self._lengths[s]} tokens: {n} cannot be taken back")
        shrunk: dict[int, list[int]] = {}
        lengths = {s: self._lengths[s] - n for s, n in counts.items()}
        for s in reversed(lengths):
            pages, kept = self._pages[s], -(-lengths[s] // self.page_size)
            if kept < len(pages):
                self._free.extend(reversed(pages[kept:]))
                shrunk[s] = pages[:kept]
        self._keep(lengths, shrunk)
        self._copy(lengths, shrunk)

    def rows(self, sequences) -> tuple[torch.Tensor, torch.Tensor]:
        """(block table, lengths) of the named sequences: the cache's own tensors where they are all, in
        order, else copies."""
        which = list(sequences)
        self._check(*which)  # (an index outside would end the process on the device)
        if which == list(range(len(self._lengths))):
            return self.block_table, self.lengths
        at = torch.tensor(which, dtype=torch.int64).to(self.lengths.device)
        return self.block_table[at], self.lengths[at]

    def free(self, *sequences: int) -> None:
        """Gives the sequences' pages back; they start anew."""
        self._check(*sequences)
        self.take_back({s: self._lengths[s] for s in reversed(sequences)})

    def _check(self, *sequences: int) -> None:
        for s in sequences:
            if not 0 <= s < len(self._lengths):
                raise ValueError(f"no sequence {s}")

    def _keep(self, lengths: dict[int, int], pages: dict[int, list[int]]) -> None:
        for s, n in lengths.items():
            self._lengths[s] = n
        for s, p in pages.items():
            self._pages[s] = p

    def _copy(self, lengths: dict[int, int], pages: dict[int, list[int]]) -> None:
        """These sequences' rows of the table and lengths, to the device: the lengths last, so that a
        failure between the two leaves no length without its pages."""
        def rows(into: torch.Tensor, values: dict) -> None:
            if values:
                at = torch.tensor(list(values)).to(into.device)
                into[at] = torch.tensor(list(values.values()), dtype=torch.int32).to(into.device)

        width = self.block_table.shape[1]
        rows(self.block_table, {s: p + [-1] * (width - len(p)) for s, p in pages.items()})
        rows(self.lengths, lengths)


class Attention(nn.Module):
    """Grouped-query attention with RMS norms of the heads and rotated positions, without biases:

        q, k, v = the heads of ``qkv_proj`` x;  norm and turn (``_lib.head_norm_rope``; v normed where
        ``v_norm``);  ``o_proj`` of softmax(scale q k^T) v over the last ``window`` (0: all) tokens

    ``scale`` is head_size^-1/2 if None.  The tables ``cos`` and ``sin`` (``rope_tables``) are the caller's:
    layers share them.  The projections are torch's products: the library has no call of a product alone
    (its own are part of the MLP's, HybridLink's and the experts' calls), and these must be differentiable."""

    def __init__(self, hidden_size: int, heads: int, kv_heads: int, head_size: int, window: int = 0,
                 scale: float | None = None, eps: float = 1e-6, v_norm: bool = True,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None) -> None:
        super().__init__()
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"heads must be a multiple of kv_heads, got {heads} and {kv_heads}")
        kw = {"dtype": dtype, "device": device}
        self.heads, self.kv_heads, self.head_size = heads, kv_heads, head_size
        self.window, self.scale, self.eps, self.v_norm = window, scale, eps, v_norm
        self.qkv_proj = nn.Linear(hidden_size, (heads + 2 * kv_heads) * head_size, bias=False, **kw)
        self.o_proj = nn.Linear(heads * head_size, hidden_size, bias=False, **kw)
        self.q_norm = nn.Parameter(torch.ones(head_size, **kw))
        self.k_norm = nn.Parameter(torch.ones(head_size, **kw))

    def _qkv(self, x: torch.Tensor):
        """The heads of x [T, hidden]: three views of one product."""
        if x.dim() != 2:
            raise ValueError(f"x must be [tokens, hidden size], got {list(x.shape)}")
        h = self.qkv_proj(x).unflatten(1, (self.heads + 2 * self.kv_heads, self.head_size))
        return h.split((self.heads, self.kv_heads, self.kv_heads), 1)

    def _out(self, o: torch.Tensor) -> torch.Tensor:
        return self.o_proj(o.flatten(1))

    def forward(self, x: torch.Tensor, positions: torch.Tensor, cu: torch.Tensor, cos: torch.Tensor,
                sin: torch.Tensor) -> torch.Tensor:
        """Packed sequences x [T, hidden], offsets ``cu``, without a cache; differentiable."""
        q, k, v = self._qkv(x)
        q, k, n = training.head_norm_rope(q, k, v if self.v_norm else None, cos, sin, positions, self.q_norm,
                                          self.k_norm, self.eps)
        return self._out(training.attention(q, k, v if n is None else n, cu, None, self.scale, True, self.window))

    @torch.no_grad()
    def prompt(self, x: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cu: torch.Tensor,
               cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor) -> torch.Tensor:
        """Packed whole prompts x [T, hidden] on their way into the cache (``positions`` and ``slots`` of
        ``PagedKVCache.append``)."""
        q, k, v = _lib.append_kv(*self._qkv(x), cos, sin, positions, slots, k_cache, v_cache, self.q_norm, self.k_norm,
                                 self.eps, v_norm=self.v_norm, return_kv=True)
        return self._out(_lib.attention(q, k, v, cu, None, self.scale, True, self.window))

    @torch.no_grad()
    def decode(self, x: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, block_table: torch.Tensor,
               lengths: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor,
               v_cache: torch.Tensor) -> torch.Tensor:
        """One new token per sequence, x [B, hidden]; ``lengths`` counts it already."""
        q = _lib.append_kv(*self._qkv(x), cos, sin, positions, slots, k_cache, v_cache, self.q_norm, self.k_norm,
                           self.eps, v_norm=self.v_norm)
        return self._out(_lib.decode_attention(q, k_cache, v_cache, block_table, lengths, self.scale, self.window))
