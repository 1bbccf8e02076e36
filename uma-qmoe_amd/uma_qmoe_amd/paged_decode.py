"""Greedy decode of several sequences together over a paged key-value cache.

``PagedDecodeGraph`` is to a batch what ``qwen_host.DecodeGraph`` is to one
sequence: one HIP graph per step of the whole model. Each layer's keys and values
lie in pages (``native_backend.KVCache``, BF16 or 8-bit floats, quantised as they
are written), which sequences of any length take from one pool as they grow and
give back when they end, and a step's attention reads what a sequence has, not what
it may have. No counterpart in the reference, whose runner
(benchmarks/runners/run_compressed_qwen_baseline.py) decodes one sequence eagerly.
"""

from __future__ import annotations

from typing import Any, Iterable

from .formats import ContractError
from .native_backend import KV_PAGE_SIZES, load_native_extension


class PagePool:
    """Which sequence has which pages (on the host). Pages are given out lowest
    first; a page belongs to one sequence at a time."""

    def __init__(self, pages: int, page_size: int, batch: int) -> None:
        self.page_size = page_size
        self.free = list(range(pages - 1, -1, -1))
        self.owned: list[list[int]] = [[] for _ in range(batch)]

    def reserve(self, lengths: Iterable[tuple[int, int]]) -> list[tuple[int, int, int]]:
        """Gives each sequence of (index, length) the pages that it lacks for
        ``length`` positions: (index, entry, page) of the new ones. Refuses, with
        nothing given, when the pool has too few."""
        missing = [(i, e) for i, n in lengths for e in range(len(self.owned[i]), -(-n // self.page_size))]
        if len(missing) > len(self.free):
            raise ContractError(f"the cache has {len(self.free)} free pages, {len(missing)} are needed")
        given = [(i, e, self.free.pop()) for i, e in missing]
        for i, _e, page in given:
            self.owned[i].append(page)
        return given

    def give_back(self, given: list[tuple[int, int, int]]) -> None:
        """Takes back what the last ``reserve`` gave."""
        for i, _e, page in reversed(given):
            self.owned[i].remove(page)
            self.free.append(page)
        self.free.sort(reverse=True)

    def release(self, index: int) -> None:
        self.free.extend(self.owned[index])
        self.free.sort(reverse=True)
        self.owned[index] = []


class PagedDecodeGraph:
    """Greedy decode of up to ``batch`` sequences of a (host) Qwen2MoE model, each
    of at most ``max_len`` positions.

    ``prefill(index, ids)`` puts a prompt into place ``index`` and chooses its first
    new token; ``extend`` adds tokens to a sequence that is there, attending to what
    the cache holds of it; ``finish`` gives its pages back. Sequences may come and go
    between steps, also after ``capture``, which records one step of the batch;
    every ``replay`` then decodes one token of each sequence. ``token`` [batch, 1]
    holds what they chose last (of places without a sequence: whatever was there),
    ``logits`` [batch, vocab] (fp32) the last step's (a replay's until the next one).
    A token is in the cache from the step on that reads it.

    Calls are made on one stream (replays of several objects, too: the library's
    workspace for the MoE blocks is one per capture stream, which objects may share).

    ``fp8_cache`` keeps keys and values in 8-bit floats (half the memory and the
    traffic). ``pages`` is the pool's size, by default enough for every sequence at
    ``max_len``; a smaller one is refused only when a step needs more than it has."""

    def __init__(self, model: Any, *, batch: int, max_len: int, page_size: int = 64, fp8_cache: bool = False,
                 pages: int | None = None) -> None:
        import torch

        self.model = model
        self.device = next(model.parameters()).device
        if self.device.type != "cuda":
            raise ContractError("a paged cache requires a HIP device")
        if getattr(model.config, "model_type", None) != "qwen2_moe":  # (others have norms of queries and keys, too)
            raise ContractError("a paged cache requires a Qwen2MoE model")
        if batch < 1 or max_len < 1:
            raise ContractError("a paged cache requires at least one sequence and one position")
        if page_size not in KV_PAGE_SIZES:
            raise ContractError(f"a paged cache has pages of {KV_PAGE_SIZES} tokens, not {page_size}")
        first = model.model.layers[0].self_attn
        if first.head_dim % 16 or first.head_dim > 256:
            raise ContractError(f"a paged cache requires heads of a multiple of 16 up to 256, not {first.head_dim}")
        self.batch, self.max_len = int(batch), int(max_len)
        width = -(-self.max_len // page_size)
        pages = self.batch * width if pages is None else int(pages)
        self.pool = PagePool(pages, page_size, self.batch)
        self.extension = load_native_extension()[1]
        self.caches = [self.extension.new_kv_cache(pages, model.config.num_key_value_heads, page_size, first.head_dim,
                                                   fp8=fp8_cache, device=self.device) for _ in model.model.layers]
        i32 = dict(dtype=torch.int32, device=self.device)
        self.page_table = torch.full((self.batch, width), -1, **i32)
        # position of the token that a sequence reads next, and the positions it then sees (-1 and 0: no sequence)
        self.positions = torch.full((self.batch,), -1, **i32)
        self.lengths = torch.zeros((self.batch,), **i32)
        self.active = torch.zeros((self.batch,), **i32)
        self.token = torch.zeros((self.batch, 1), dtype=torch.long, device=self.device)
        self.next_positions: list[int | None] = [None] * self.batch  # host copy of ``positions``
        self.logits = None
        self.graph = None
        self._graph_logits = None  # what a replay writes
        self.stream = torch.cuda.Stream(device=self.device)  # warm-up and capture, as DecodeGraph

    # ------------------------------------------------------------- the model --
    def _forward(self, input_ids: Any, position_ids: Any, attend: Any) -> Any:
        """Logits of the last position (fp32 [rows, vocab]); ``attend(layer index,
        attention module, q, k, v)`` gives [rows, tokens, heads * head_dim]."""
        from transformers.models.qwen2_moe.modeling_qwen2_moe import apply_rotary_pos_emb

        inner = self.model.model
        hidden = inner.embed_tokens(input_ids)
        cos, sin = inner.rotary_emb(hidden, position_ids)
        for i, layer in enumerate(inner.layers):
            attn = layer.self_attn
            x = layer.input_layernorm(hidden)
            shape = (*x.shape[:-1], -1, attn.head_dim)
            q, k, v = (p(x).view(shape).transpose(1, 2) for p in (attn.q_proj, attn.k_proj, attn.v_proj))
            q, k = apply_rotary_pos_emb(q, k, cos, sin)
            hidden = hidden + attn.o_proj(attend(i, attn, q, k, v))
            hidden = hidden + layer.mlp(layer.post_attention_layernorm(hidden))
        return self.model.lm_head(inner.norm(hidden[:, -1:]))[:, -1].float()

    @staticmethod
    def _dense(attn: Any, q: Any, k: Any, v: Any, start: int, window: int | None) -> Any:
        """Attention of new tokens at positions ``start`` on over positions from 0."""
        import torch
        from torch.nn.attention import SDPBackend, sdpa_kernel

        n, total = q.shape[2], k.shape[2]
        share = q.shape[1] // k.shape[1]
        if share > 1:
            k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
        mask = None
        if start or (window is not None and window < total):
            at = torch.arange(start, total, device=q.device)[:, None]
            seen = torch.arange(total, device=q.device)
            mask = seen <= at
            if window is not None:
                mask &= seen > at - window
        with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
            out = torch.nn.functional.scaled_dot_product_attention(q, k.contiguous(), v.contiguous(), attn_mask=mask,
                                                                   is_causal=mask is None, scale=attn.scaling)
        return out.transpose(1, 2).reshape(q.shape[0], n, -1)

    # --------------------------------------------------------- the sequences --
    def _place(self, index: int) -> int:
        if not 0 <= index < self.batch:
            raise ContractError(f"no place {index} in a batch of {self.batch}")
        return index

    def _count(self, ids: Any) -> int:
        """How many tokens ``ids`` has, which must be [1, n] ids on the device."""
        import torch

        if not torch.is_tensor(ids) or ids.ndim != 2 or ids.shape[0] != 1 or ids.dtype not in (torch.long, torch.int32):
            raise ContractError("a sequence takes a tensor of [1, n] token ids (int64 or int32)")
        if ids.device != self.device:
            raise ContractError(f"a sequence takes token ids on {self.device}, not on {ids.device}")
        return int(ids.shape[1])

    def _enter(self, given: list[tuple[int, int, int]]) -> None:
        for i, entry, page in given:
            self.page_table[i, entry] = page

    def finish(self, index: int) -> None:
        """Ends the sequence at ``index`` (if there is one): its pages are free for others."""
        self.pool.release(self._place(index))
        self.page_table[index] = -1
        self.positions[index] = -1
        self.lengths[index] = 0
        self.active[index] = 0
        self.next_positions[index] = None

    def prefill(self, index: int, prompt_ids: Any) -> Any:
        """Starts a sequence at ``index`` (ending the one there) with a prompt of
        [1, n] token ids on the device; returns its first new token [1, 1]. If the
        model fails the place is empty."""
        self._place(index)
        n = self._count(prompt_ids)
        if n < 1 or n >= self.max_len:
            raise ContractError("prompt must be non-empty and shorter than the cache")
        missing = -(-n // self.pool.page_size) - len(self.pool.owned[index])
        if missing > len(self.pool.free):
            raise ContractError(f"the cache has {len(self.pool.free)} free pages, {missing} are needed")
        self.finish(index)
        return self._grow(index, 0, prompt_ids)

    def extend(self, index: int, ids: Any) -> Any:
        """Adds tokens ([1, n] ids on the device) behind those that the cache holds
        of the sequence at ``index``, and chooses the next one [1, 1]. The token
        that was chosen last is not in the cache yet: it stays in the sequence as
        the first of ``ids``, or not at all. If the model fails the sequence is as
        it was."""
        start, n = self.next_positions[self._place(index)], self._count(ids)
        if start is None:
            raise ContractError(f"no sequence at {index} to add tokens to: prefill() one")
        if n < 1 or start + n >= self.max_len:
            raise ContractError("a sequence must grow by at least one token and stay shorter than the cache")
        return self._grow(index, start, ids)

    def _grow(self, index: int, start: int, ids: Any) -> Any:
        """Tokens at positions ``start`` on of the sequence at ``index``, and the next choice."""
        import torch

        n = ids.shape[1]
        given = self.pool.reserve([(index, start + n)])
        table = self.page_table[index:index + 1]

        def attend(i: int, attn: Any, q: Any, k: Any, v: Any) -> Any:
            past = self.extension.kv_read(self.caches[i], table, starts, start) if start else None
            self.extension.kv_append(self.caches[i], k, v, table, starts)
            if past is not None:
                k, v = torch.cat([past[0], k], 2), torch.cat([past[1], v], 2)
            return self._dense(attn, q, k, v, start, getattr(attn, "sliding_window", None))

        try:
            self._enter(given)
            starts = torch.full((1,), start, dtype=torch.int32, device=self.device)
            with torch.no_grad():
                logits = self._forward(ids, torch.arange(start, start + n, device=self.device)[None], attend)
                self.token[index] = logits[0].argmax()
        except BaseException:
            # (what was written lies behind the sequence's end, where nothing is read)
            table[0, len(self.pool.owned[index]) - len(given):] = -1
            self.pool.give_back(given)
            raise
        self.positions[index] = start + n
        self.lengths[index] = start + n + 1
        self.active[index] = 1
        self.next_positions[index] = start + n
        return self.token[index:index + 1].clone()

    # ------------------------------------------------------------- the steps --
    def _step(self) -> Any:
        import torch

        def attend(i: int, attn: Any, q: Any, k: Any, v: Any) -> Any:
            self.extension.kv_append(self.caches[i], k, v, self.page_table, self.positions)
            out = self.extension.paged_attention(q[:, :, 0], self.caches[i], self.page_table, self.lengths,
                                                 scale=attn.scaling, window=getattr(attn, "sliding_window", None))
            return out.reshape(self.batch, 1, -1)

        logits = self._forward(self.token, self.positions.clamp_min(0)[:, None].long(), attend)
        self.token.copy_(torch.where(self.active[:, None] != 0, logits.argmax(-1, keepdim=True), self.token))
        self.positions.add_(self.active)
        self.lengths.add_(self.active)
        return logits

    def _prepare_step(self) -> None:
        """Pages for every sequence's next position, or a refusal with nothing changed."""
        if all(p is None for p in self.next_positions):
            raise ContractError("no sequence to decode")
        full = [i for i, p in enumerate(self.next_positions) if p is not None and p >= self.max_len]
        if full:
            raise ContractError(f"sequences {full} have filled their places in the cache: finish() them first")
        self._enter(self.pool.reserve((i, p + 1) for i, p in enumerate(self.next_positions) if p is not None))

    def _advance(self) -> None:
        self.next_positions = [p if p is None else p + 1 for p in self.next_positions]

    def step_eager(self) -> Any:
        """One token of each sequence without the graph (the same operations)."""
        import torch

        self._prepare_step()
        with torch.no_grad():
            self.logits = self._step()
        self._advance()
        return self.token.clone()

    def capture(self) -> None:
        """Records one step. A warm-up step runs before it on the capture's stream
        (it writes the sequences' next positions, which the next step writes
        again); the tokens and positions are put back afterwards. ``logits`` stay
        those of the last step: recording computes none."""
        import torch

        self._prepare_step()
        counters = (self.token, self.positions, self.lengths)
        saved = [c.clone() for c in counters]
        self.stream.wait_stream(torch.cuda.current_stream(self.device))
        with torch.no_grad(), torch.cuda.stream(self.stream):
            self._step()
            for c, v in zip(counters, saved):
                c.copy_(v)
        torch.cuda.current_stream(self.device).wait_stream(self.stream)
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph, stream=self.stream):
            logits = self._step()
        self.graph, self._graph_logits = graph, logits

    def replay(self) -> Any:
        """One token of each sequence: the token buffer (device, [batch, 1]) after the step."""
        if self.graph is None:
            raise ContractError("capture() a decode step first")
        self._prepare_step()
        self.graph.replay()
        self.logits = self._graph_logits
        self._advance()
        return self.token


__all__ = ["PagePool", "PagedDecodeGraph"]
