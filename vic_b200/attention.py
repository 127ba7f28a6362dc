"""The latent-attention sublayer of a decode layer, and the layer made of it and the MoE sublayer.

The reference runs this sublayer token by token over a flat cache (src/runtime/attention.rs; kernels cuda/src/kernels.cu:1570-1740).
Here the newest tokens of a batch go through it together: ``LatentCache`` keeps the paged rows of every layer and, per step, where the new
tokens' rows go; ``LatentAttention`` is one layer's weights and its launches; ``DecodeLayer`` puts it before MoeDecoder or
GroupedDecoder.  Projections from and to the hidden state are plain library products.  After ``LatentCache.begin_step`` (host) everything
is device work on fixed buffers and can be captured into a CUDA graph."""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from . import kernels
from .core_types import LatentShape
from .kernels import LATENT_RANK, LATENT_ROPE, LATENT_ROW
from .lib import Vib3Error


class LatentCache:
    """Paged latent rows of ``layers`` layers for up to ``max_sequences`` sequences of up to ``max_pages`` pages each.  One page table
    serves all layers.  Device buffers of a step (fixed addresses): ``table``, ``lens``, ``positions`` and ``slots`` (behind the step's rows: 0
    and -1).  A captured step is for steps of its own q_len: with fewer new tokens per sequence give ``begin_step`` that q_len."""

    def __init__(self, layers: int, pages: int, page_size: int, max_sequences: int, max_pages: int, dtype: torch.dtype, device,
                 max_tokens: int = 128):
        if page_size <= 0 or page_size % 8:
            raise ValueError("page_size: a positive multiple of 8")
        if max_tokens < max_sequences:
            raise ValueError("max_tokens: at least one token per sequence")
        self.page_size, self.max_sequences, self.max_pages, self.max_tokens = page_size, max_sequences, max_pages, max_tokens
        self.rows = torch.zeros(layers, pages, page_size, LATENT_ROW, dtype=dtype, device=device)
        self.table = torch.zeros(max_sequences, max_pages, dtype=torch.int32, device=device)
        self._host_table = torch.zeros(max_sequences, max_pages, dtype=torch.int32)     # (only new pages change it: most steps bring none)
        self._table_changed = False
        self.lens = torch.zeros(max_sequences, dtype=torch.int32, device=device)
        self.positions = torch.zeros(max_tokens, dtype=torch.int32, device=device)
        self.slots = torch.full((max_tokens,), -1, dtype=torch.int64, device=device)
        self.host_lens: List[int] = [0] * max_sequences
        self.step_rows = 0      # rows of the step that the buffers describe
        self._pages_of: List[List[int]] = [[] for _ in range(max_sequences)]
        self._free = list(range(pages - 1, -1, -1))

    def begin_step(self, new_tokens: Sequence[int], q_len: Optional[int] = None) -> None:
        """Sequence b gets new_tokens[b] tokens (0: none): pages for them, their positions and slots, the lengths with them.
        A step's rows are q_len (default: the largest count) per sequence, the new tokens last.  The rows before them are padding: nothing is
        stored of them, but they attend to what their sequence has (and so cost its cache's bytes), and what comes of them means nothing."""
        if len(new_tokens) != self.max_sequences:
            raise ValueError(f"{self.max_sequences} counts expected")
        q_len = max(new_tokens) if q_len is None else q_len
        if min(new_tokens) < 0 or max(new_tokens) > q_len or q_len * self.max_sequences > self.max_tokens:
            raise ValueError("counts have to lie in 0 .. q_len, and q_len * sequences within max_tokens")
        need = [-(-(n + k) // self.page_size) for n, k in zip(self.host_lens, new_tokens)]
        if max(need) > self.max_pages or sum(max(0, n - len(p)) for n, p in zip(need, self._pages_of)) > len(self._free):
            raise Vib3Error("latent cache: no page left for the step's tokens", -8)
        positions, slots = [], []
        for b, k in enumerate(new_tokens):
            own, first = self._pages_of[b], self.host_lens[b]
            while len(own) < need[b]:
                own.append(self._free.pop())
                self._host_table[b, len(own) - 1] = own[-1]
                self._table_changed = True
            pad = q_len - k
            positions += [0] * pad + list(range(first, first + k))
            slots += [-1] * pad + [own[p // self.page_size] * self.page_size + p % self.page_size for p in range(first, first + k)]
            self.host_lens[b] = first + k
        n, older = len(positions), self.step_rows
        if n < older:       # a captured step of more rows than this one finds no slots behind it
            self.positions[n:older].zero_()
            self.slots[n:older].fill_(-1)
        self.step_rows = n
        self.positions[:n].copy_(torch.tensor(positions, dtype=torch.int32))
        self.slots[:n].copy_(torch.tensor(slots, dtype=torch.int64))
        if self._table_changed:
            self.table.copy_(self._host_table)      # (from pageable memory: read before the call returns)
            self._table_changed = False
        self.lens.copy_(torch.tensor(self.host_lens, dtype=torch.int32))

    def release(self, sequence: int) -> None:
        """Forget a sequence; its pages may go to others."""
        self._free += self._pages_of[sequence][::-1]
        self._host_table[sequence] = 0
        self._table_changed = True
        self._pages_of[sequence] = []
        self.host_lens[sequence] = 0


class LatentAttention:
    """One layer: x [T, hidden] -> output [T, hidden], T = sequences * q_len rows in the cache's order.

    ``w_q`` [heads * (nope + 64), hidden], ``w_kv`` [576, hidden], ``kv_norm`` [512], ``kv_b`` [heads, nope + value, 512] (the heads' key
    and value matrices), ``w_o`` [hidden, heads * value]; one dtype, fp16 or bf16.  ``inv_freq`` [32] float64: the angles per position, where
    they are not the powers of the shape's rope_theta.  Queries of low rank: ``q_down`` [q_rank, hidden] and ``q_norm`` [q_rank], and ``w_q``
    [heads * (nope + 64), q_rank] then takes norm(x q_down^T)."""

    def __init__(self, shape: LatentShape, w_q: torch.Tensor, w_kv: torch.Tensor, kv_norm: torch.Tensor, kv_b: torch.Tensor,
                 w_o: torch.Tensor, max_tokens: int = 128, workspace: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
                 q_down: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None):
        dev, dt, H = w_q.device, w_q.dtype, shape.heads
        if (q_down is None) != (q_norm is None):
            raise ValueError("q_down and q_norm: both or neither")
        q_width = shape.hidden
        if q_down is not None:
            if q_down.dim() != 2 or q_down.shape[1] != shape.hidden or q_down.dtype != dt or q_down.device != dev:
                raise ValueError(f"q_down: [q_rank, {shape.hidden}] of the layer's dtype on {dev} expected")
            q_width = q_down.shape[0]
            if q_norm.shape != (q_width,) or q_norm.dtype not in (torch.float16, torch.bfloat16) or not q_norm.is_contiguous() or q_norm.device != dev:
                raise ValueError(f"q_norm: contiguous fp16 or bf16 [{q_width}] on {dev} expected")
            self.q_low32 = torch.zeros(max_tokens, q_width, device=dev)
            self.q_low = torch.zeros(max_tokens, q_width, dtype=dt, device=dev)
        self.q_down, self.q_norm = q_down, q_norm
        if w_q.shape != (H * (shape.nope + LATENT_ROPE), q_width) or w_kv.shape != (LATENT_ROW, shape.hidden) or kv_norm.shape != (LATENT_RANK,) or \
                kv_b.shape != (H, shape.nope + shape.value, LATENT_RANK) or w_o.shape != (shape.hidden, H * shape.value):
            raise ValueError("weights do not have the layer's shape")
        self.shape, self.max_tokens = shape, max_tokens
        self.w_q, self.w_kv, self.kv_norm, self.kv_b, self.w_o = w_q, w_kv, kv_norm, kv_b, w_o
        if inv_freq is None:
            inv_freq = shape.rope_theta ** (-torch.arange(0, LATENT_ROPE, 2, dtype=torch.float64, device=dev) / LATENT_ROPE)
        elif inv_freq.shape != (LATENT_ROPE // 2,) or inv_freq.dtype != torch.float64 or inv_freq.device != dev or not inv_freq.is_contiguous():
            raise ValueError(f"inv_freq: contiguous float64 [32] on {dev} expected")
        self.inv_freq = inv_freq
        self.q_in = torch.zeros(max_tokens, H * (shape.nope + LATENT_ROPE), dtype=dt, device=dev)
        self.kv_in = torch.zeros(max_tokens, LATENT_ROW, dtype=dt, device=dev)
        self.q = torch.zeros(max_tokens, H, LATENT_ROW, dtype=dt, device=dev)
        self.o = torch.zeros(max_tokens, H, LATENT_RANK, dtype=dt, device=dev)
        self.v = torch.zeros(max_tokens, H, shape.value, dtype=dt, device=dev)
        self.out = torch.zeros(max_tokens, shape.hidden, dtype=dt, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        # layers that run one after another may share it
        self.workspace = torch.empty(kernels.latent_attention_workspace_bytes(), dtype=torch.uint8, device=dev) if workspace is None else workspace

    def check_rows(self, rows: int, cache: LatentCache) -> None:
        if rows > self.max_tokens or rows != cache.step_rows:
            raise ValueError(f"the step's {cache.step_rows} rows (sequences * q_len) expected, at most {self.max_tokens}; got {rows}")

    def forward(self, x: torch.Tensor, cache: LatentCache, layer: int) -> torch.Tensor:
        """The step that ``cache.begin_step`` laid out.  Returns a view of ``self.out``."""
        sh, T = self.shape, x.shape[0]
        self.check_rows(T, cache)
        if T == 0:
            return self.out[:0]
        rows, pos = cache.rows[layer], cache.positions[:T]
        torch.matmul(x, self.w_kv.t(), out=self.kv_in[:T])
        q = x
        if self.q_down is not None:
            q = torch.matmul(x, self.q_down.t(), out=self.q_low[:T])
            self.q_low32[:T].copy_(q)
            kernels.residual_rms_norm(self.q_low32[:T], None, self.q_norm, sh.eps, q)
        torch.matmul(q, self.w_q.t(), out=self.q_in[:T])
        kernels.latent_append(self.kv_in[:T], self.kv_norm, sh.eps, pos, cache.slots[:T], self.inv_freq, rows,
                              pairs=sh.pairs, rope_scale=sh.rope_scale, status=self.status)
        kernels.latent_query(self.q_in[:T].view(T, sh.heads, sh.nope + LATENT_ROPE), self.kv_b[:, :sh.nope], pos, self.inv_freq, self.q[:T],
                             pairs=sh.pairs, rope_scale=sh.rope_scale, status=self.status)
        kernels.latent_attention(self.q[:T], rows, cache.table, cache.lens, sh.scale, self.o[:T], workspace=self.workspace, status=self.status)
        kernels.latent_value(self.o[:T], self.kv_b[:, sh.nope:], self.v[:T], status=self.status)
        torch.matmul(self.v[:T].view(T, sh.heads * sh.value), self.w_o.t(), out=self.out[:T])
        return self.out[:T]


class DecodeLayer:
    """h += attention(norm(h)), h += moe(norm(h)) for a step's rows: ``moe`` is a MoeDecoder (one row) or a GroupedDecoder.
    The norms' weights [hidden] are fp16 or bf16.  ``selection_bias`` [experts] fp32 is added to the router's scores for the selection only."""

    def __init__(self, attention: LatentAttention, moe, layer: int, attention_norm: torch.Tensor, moe_norm: torch.Tensor, eps: float = 1e-6,
                 selection_bias: Optional[torch.Tensor] = None):
        hidden, dev = attention.shape.hidden, attention.w_q.device
        for norm in (attention_norm, moe_norm):
            if norm.shape != (hidden,) or norm.dtype not in (torch.float16, torch.bfloat16) or not norm.is_contiguous() or norm.device != dev:
                raise ValueError(f"norm weights: contiguous fp16 or bf16 [{hidden}] on {dev} expected")
        if moe.model.shape.hidden != hidden or not -moe.model.n_layers <= layer < moe.model.n_layers or moe.model.router_w.device != dev:
            raise ValueError(f"moe: a decoder on {dev} with layer {layer} and rows of {hidden} values expected")
        if selection_bias is not None and (selection_bias.shape != (moe.model.shape.num_experts,) or selection_bias.dtype != torch.float32
                                           or not selection_bias.is_contiguous() or selection_bias.device != dev):
            raise ValueError(f"selection_bias: contiguous fp32 [{moe.model.shape.num_experts}] on {dev} expected")
        self.selection_bias = selection_bias
        self.attention, self.moe, self.layer = attention, moe, layer
        self.moe_rows = getattr(moe, "max_tokens", 1)       # of a GroupedDecoder; a MoeDecoder takes one row
        self.attention_norm, self.moe_norm, self.eps = attention_norm, moe_norm, eps
        self.x = torch.zeros(attention.max_tokens, attention.shape.hidden, dtype=attention.w_q.dtype, device=attention.w_q.device)

    def forward(self, h: torch.Tensor, cache: LatentCache) -> torch.Tensor:
        """h [T, hidden] fp32, updated in place.  Rows, types and decoders that do not fit are refused before h or the cache has changed."""
        hidden = self.attention.shape.hidden
        if h.dim() != 2 or h.shape[1] != hidden or h.dtype != torch.float32 or h.stride(1) != 1 or h.stride(0) < hidden:
            raise ValueError(f"h: fp32 [T, {hidden}] with contiguous rows expected")
        if h.device != self.x.device or (h.is_cuda and h.get_device() != torch.cuda.current_device()):
            raise ValueError(f"h: on the layer's device ({self.x.device}), which has to be the current one, expected; got {h.device}")
        T = h.shape[0]
        self.attention.check_rows(T, cache)
        if T > self.moe_rows:
            raise ValueError(f"the MoE decoder takes {self.moe_rows} row(s), got {T} (MoeDecoder takes one; GroupedDecoder takes several)")
        if not -cache.rows.shape[0] <= self.layer < cache.rows.shape[0]:
            raise ValueError(f"cache: {cache.rows.shape[0]} layers, none with number {self.layer}")
        if T == 0:
            return h
        x = self.x[:T]
        kernels.residual_rms_norm(h, None, self.attention_norm, self.eps, x)
        delta = self.attention.forward(x, cache, self.layer)
        kernels.residual_rms_norm(h, delta, self.moe_norm, self.eps, x, early_dependents=True)
        if hasattr(self.moe, "max_tokens"):
            self.moe.forward(self.layer, x, out=h, accumulate=True, hold=True, bias=self.selection_bias)
        else:
            self.moe.forward_layer(self.layer, x[0], out=h[0], accumulate=True, bias=self.selection_bias, hold=True)
        return h
