"""Device-resident recurrent state carried between tokens and loop passes.

Mirrors RecurrentState (model/recurrent_state.py:76-98): per loop pass and
block, keyed ``"loop{i}.core.{j}"`` exactly as PhysicalBlock builds its state
keys (model/model.py:168-171) —
  * ``gdn_states[key]``         [B, H, K, V] fp32 delta-rule state
  * ``gdn_conv_histories[key]`` [B, 3, D] bf16, last three GDN block inputs
  * ``local_k[key]`` / ``local_v[key]``  ring caches [B, W, H*Dh] / [B, W, D]
    of the CSA window (token p at slot p % W).  The reference keeps the
    normed hidden rows and re-projects K/V every step (csa.py:176-178); the
    cache holds the same projections computed once.
  * ``router_latents[key]``    [B, W, L] fp32 ring of the router's LayerNorm'd
    MLA latents of the last W positions (router_latent_histories,
    model/model.py:239-247; only with the router's local context).
  * CSA remote branch (only with ``csa_compression``): ``remote_k[key]``
    [B, C, H*Dh] / ``remote_v[key]`` [B, C, D] bf16, the keys and values of
    the row's completed block summaries (compressed memory keys / values,
    csa.py:208-256), ``remote_count[key]`` [B] int32 how many there are,
    ``remote_sum[key]`` [B, D] fp32 / ``remote_pending[key]`` [B] int32 the
    pending partial block (MemoryState.pending_sum / pending_count).  C =
    ceil(max_len / ratio) summaries.  The reference also appends an
    invisible entry for every decode token that completes no block; no query
    can see those, so they are not kept.
  * ``local_vo[key]`` [B, W, D] bf16: the CSA value ring folded with the
    block's output projection (W_o v), kept by the batch-1 persistent decode
    step (persistent.py) once ``folded_rings`` is set; the plain ``local_v``
    then falls behind until the next prefill.
  * ``positions`` [B] int32, position of the next token of each row.
All buffers are allocated once for a batch size so that a captured decode
graph can update them in place.
"""
from __future__ import annotations

import torch

from .config import HybridConfig


def state_key(loop: int, block: int) -> str:
    return f"loop{loop}.core.{block}"


class RecurrentState:
    def __init__(self, cfg: HybridConfig, batch: int, device: torch.device | str = "cuda",
                 max_len: int = 8192):
        """max_len: the longest sequence (prompt + generated tokens) the CSA
        remote branch's summary memory holds."""
        self.cfg = cfg
        self.batch = int(batch)
        self.max_len = int(max_len)
        self.device = torch.device(device)
        d = cfg.d_model
        self.gdn_states: dict[str, torch.Tensor] = {}
        self.gdn_conv_histories: dict[str, torch.Tensor] = {}
        self.local_k: dict[str, torch.Tensor] = {}
        self.local_v: dict[str, torch.Tensor] = {}
        for i in range(cfg.num_loops):
            for j in range(cfg.n_blocks):
                key = state_key(i, j)
                if cfg.block_kind(j) == "gdn":
                    self.gdn_states[key] = torch.zeros(
                        batch, cfg.gdn_heads, cfg.gdn_key_dim, cfg.gdn_value_dim,
                        dtype=torch.float32, device=self.device)
                    self.gdn_conv_histories[key] = torch.zeros(
                        batch, cfg.conv_kernel - 1, d, dtype=torch.bfloat16, device=self.device)
                else:
                    self.local_k[key] = torch.zeros(
                        batch, cfg.csa_window, cfg.csa_heads * cfg.csa_head_dim,
                        dtype=torch.bfloat16, device=self.device)
                    self.local_v[key] = torch.zeros(batch, cfg.csa_window, d,
                                                    dtype=torch.bfloat16, device=self.device)
        # router local context: the LayerNorm'd latents of the last W positions
        # (position p at slot p % W) per loop and block
        self.router_latents: dict[str, torch.Tensor] = {}
        if cfg.router_context:
            for i in range(cfg.num_loops):
                for j in range(cfg.n_blocks):
                    self.router_latents[state_key(i, j)] = torch.zeros(
                        batch, cfg.router_local_context, cfg.router_latent_dim,
                        dtype=torch.float32, device=self.device)
        self.remote_k: dict[str, torch.Tensor] = {}
        self.remote_v: dict[str, torch.Tensor] = {}
        self.remote_count: dict[str, torch.Tensor] = {}
        self.remote_sum: dict[str, torch.Tensor] = {}
        self.remote_pending: dict[str, torch.Tensor] = {}
        if cfg.csa_compression:
            cap = -(-self.max_len // cfg.csa_compression)
            hd = cfg.csa_heads * cfg.csa_head_dim
            for key in self.local_k:
                self.remote_k[key] = torch.zeros(batch, cap, hd, dtype=torch.bfloat16,
                                                 device=self.device)
                self.remote_v[key] = torch.zeros(batch, cap, d, dtype=torch.bfloat16,
                                                 device=self.device)
                self.remote_count[key] = torch.zeros(batch, dtype=torch.int32, device=self.device)
                self.remote_sum[key] = torch.zeros(batch, d, dtype=torch.float32,
                                                   device=self.device)
                self.remote_pending[key] = torch.zeros(batch, dtype=torch.int32,
                                                       device=self.device)
        self.local_vo: dict[str, torch.Tensor] = {}
        self.folded_rings = False
        self.positions = torch.zeros(batch, dtype=torch.int32, device=self.device)

    def _tables(self):
        return (("gdn_states", self.gdn_states), ("gdn_conv_histories", self.gdn_conv_histories),
                ("local_k", self.local_k), ("local_v", self.local_v),
                ("router_latents", self.router_latents), ("remote_k", self.remote_k),
                ("remote_v", self.remote_v), ("remote_count", self.remote_count),
                ("remote_sum", self.remote_sum), ("remote_pending", self.remote_pending),
                ("local_vo", self.local_vo))

    def fill_synthetic(self, position: int, seed: int = 0) -> None:
        """Stand-in for a prefilled context of `position` tokens (benchmarks
        whose cost does not depend on the context's values): ring caches and
        conv histories ~ N(0, 1), GDN states ~ N(0, 0.05), positions =
        position.  Drawn on the device from a seeded generator."""
        g = torch.Generator(device=self.device)
        g.manual_seed(int(seed))
        for t in (*self.local_k.values(), *self.local_v.values(),
                  *self.gdn_conv_histories.values()):
            t.copy_(torch.randn(t.shape, generator=g, device=self.device, dtype=torch.float32))
        for t in self.gdn_states.values():
            t.normal_(0.0, 0.05, generator=g)
        self.positions.fill_(int(position))

    def reset_rows(self, rows: torch.Tensor) -> None:
        """Clear the state of the selected rows (recurrent_state.py:218-244)."""
        mask = rows.to(device=self.device, dtype=torch.bool)
        for t in (*self.gdn_states.values(), *self.gdn_conv_histories.values(),
                  *self.router_latents.values(), *self.remote_count.values(),
                  *self.remote_sum.values(), *self.remote_pending.values()):
            t[mask] = 0
        self.positions[mask] = 0

    def zero_(self) -> None:
        """Zero every state tensor and position (a fresh conversation); on a
        CUDA device one native launch over a table of the tensors' regions,
        built on the first call (make that call before capturing it in a CUDA
        graph) and rebuilt when a table's tensors change."""
        tensors = [t for _, table in self._tables() for t in table.values()] + [self.positions]
        if self.device.type != "cuda":
            for t in tensors:
                t.zero_()
            return
        from . import kernels
        key = tuple((t.data_ptr(), t.numel() * t.element_size()) for t in tensors)
        if getattr(self, "_zero_key", None) != key:
            self._zero_table, self._zero_max = kernels.region_table(tensors, self.device)
            self._zero_key = key
        kernels.zero_regions(self._zero_table, self._zero_max)

    def nbytes(self) -> int:
        tensors = [t for _, table in self._tables() for t in table.values()] + [self.positions]
        return sum(t.numel() * t.element_size() for t in tensors)

    def state_dict(self) -> dict[str, torch.Tensor]:
        out: dict[str, torch.Tensor] = {"positions": self.positions.clone(),
                                        "folded_rings": torch.tensor(self.folded_rings)}
        for name, table in self._tables():
            for key, t in table.items():
                out[f"{name}.{key}"] = t.clone()
        return out

    def load_state_dict(self, sd: dict[str, torch.Tensor]) -> None:
        """Tables missing from `sd` (the folded rings of a state saved before
        the persistent step created them) keep their contents."""
        self.positions.copy_(sd["positions"])
        self.folded_rings = bool(sd.get("folded_rings", torch.tensor(False)))
        for name in sd:  # folded rings this state has not created yet
            key = name[len("local_vo."):]
            if name.startswith("local_vo.") and key not in self.local_vo:
                self.local_vo[key] = torch.empty_like(self.local_v[key])
        for name, table in self._tables():
            for key, t in table.items():
                if name == "local_vo" and f"{name}.{key}" not in sd:
                    continue
                t.copy_(sd[f"{name}.{key}"])


class PagedKVCache:
    """Keys and values of attention blocks that reach further than a ring of
    ``csa_window`` rows: pages of ``page_size`` positions handed out to the rows
    of a batch as they grow, so rows of any lengths share one memory.

      * ``k[layer]`` / ``v[layer]`` [pages, kv_heads, page_size, head_dim] (bf16 or fp16)
      * ``block_table`` [batch, max_pages] int32, the pages of every row (-1: none)
      * ``lengths`` [batch] int32, positions of every row
    One table serves all layers.  Pages are managed on the host (``reserve``,
    ``extend``, ``release``); ``append`` and ``attend`` are the kernels of
    kernels.py on one layer.

    A decode step captured in a CUDA graph counts ``lengths`` up inside the graph
    (``lengths.add_(live)``, live [batch] int32: 1 for the rows that go on, 0 for
    released ones).  Its pages are reserved before the replays, and ``advance``
    tells the host afterwards how many tokens they added: the device's lengths
    are never overwritten by the host's, and pages are handed out by the host's.
    """

    def __init__(self, kv_heads: int, head_dim: int, *, batch: int, pages: int,
                 page_size: int = 64, max_pages: int | None = None, layers: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        """max_pages: pages of one row at most (default: all of them)."""
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError("page_size must be 16, 32, 64, 128 or 256")
        if head_dim not in (64, 128) or dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("head dimensions 64 and 128 in bf16 or fp16 are served")
        if kv_heads < 1 or batch < 1 or pages < 1 or layers < 1:
            raise ValueError("kv_heads, batch, pages and layers must be positive")
        self.batch, self.page_size = int(batch), int(page_size)
        self.max_pages = int(pages if max_pages is None else max_pages)
        self.device = torch.device(device)
        shape = (int(pages), int(kv_heads), self.page_size, int(head_dim))
        self.k = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(layers)]
        self.block_table = torch.full((self.batch, self.max_pages), -1, dtype=torch.int32,
                                      device=self.device)
        self.lengths = torch.zeros(self.batch, dtype=torch.int32, device=self.device)
        self._held: list[list[int]] = [[] for _ in range(self.batch)]
        self._length = [0] * self.batch
        self._free = list(range(int(pages) - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _counts(self, tokens) -> list[int]:
        counts = [int(t) for t in tokens]
        if len(counts) != self.batch or min(counts) < 0:
            raise ValueError(f"one count >= 0 for each of the {self.batch} rows is needed")
        return counts

    def reserve(self, tokens) -> None:
        """Pages for tokens[b] more positions of every row; lengths stay.  Raises
        and changes nothing where pages run out or a row outgrows max_pages."""
        counts = self._counts(tokens)
        more = [max(0, -(-(n + c) // self.page_size) - len(h))
                for n, c, h in zip(self._length, counts, self._held)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(more)} are needed")
        if any(len(h) + m > self.max_pages for h, m in zip(self._held, more)):
            raise RuntimeError(f"a row has at most {self.max_pages} pages")
        for b, m in enumerate(more):
            if m:
                first = len(self._held[b])
                self._held[b] += [self._free.pop() for _ in range(m)]
                self.block_table[b, first:first + m] = torch.tensor(
                    self._held[b][first:], dtype=torch.int32).to(self.device)

    def extend(self, tokens) -> torch.Tensor:
        """Reserves the pages and counts the lengths up, the host's and the
        device's; returns cu_q [batch + 1] int32, the packing of the new tokens."""
        counts = self._counts(tokens)
        self.reserve(counts)
        self._length = [n + c for n, c in zip(self._length, counts)]
        cu_q = torch.tensor([0, *counts], dtype=torch.int64).cumsum(0).to(torch.int32).to(self.device)
        self.lengths.add_(cu_q[1:] - cu_q[:-1])
        return cu_q

    def advance(self, tokens) -> None:
        """Counts the host's lengths up by tokens that captured steps have already
        counted on the device.  Raises and changes nothing where a row would
        outgrow its reserved pages (its last tokens were not stored)."""
        counts = self._counts(tokens)
        length = [n + c for n, c in zip(self._length, counts)]
        for b, (n, held) in enumerate(zip(length, self._held)):
            if n > len(held) * self.page_size:
                raise RuntimeError(f"row {b} has {len(held)} pages reserved, {n} positions need more")
        self._length = length

    def release(self, rows) -> None:
        """Gives the pages of the rows back; their lengths are 0.  Raises and changes
        nothing where a row is none of the batch's."""
        rows = {int(r) for r in rows}
        if any(r < 0 or r >= self.batch for r in rows):
            raise ValueError(f"rows 0 .. {self.batch - 1} can be released")
        for b in rows:
            self._free += reversed(self._held[b])
            self._held[b], self._length[b] = [], 0
            self.block_table[b].fill_(-1)
            self.lengths[b] = 0

    def append(self, layer: int, q, k, v, cu_q=None, **options) -> torch.Tensor:
        """kernels.paged_append on a layer: the new tokens' keys and values into
        their pages, the queries back.  cu_q of extend; None: one token per row."""
        from . import kernels
        return kernels.paged_append(q, k, v, self.k[layer], self.v[layer], self.block_table,
                                    self.lengths, cu_q=cu_q, **options)

    def attend(self, layer: int, q, cu_q=None, **options) -> torch.Tensor:
        """Attention of the new tokens over their rows: kernels.paged_prefill, or
        kernels.paged_decode where cu_q is None (one token per row)."""
        from . import kernels
        at = (self.k[layer], self.v[layer], self.block_table, self.lengths)
        if cu_q is None:
            return kernels.paged_decode(q, *at, **options)
        return kernels.paged_prefill(q, *at, cu_q, **options)
