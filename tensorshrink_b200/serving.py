"""A Llama-shaped decoder served from 4-bit floating-point or 8-bit integer
projections and a paged key-value cache of 16 or 8 bits: `fp4_linear` or
`int8_linear`, `qk_norm_rope`, `paged_append`, `paged_decode_attention` and
`paged_evict`, `paged_reserve` and `paged_release`, as a serving program strings them
together.

`decoder.QuantDecoder` decodes a batch whose sequences all stand at one
position of a dense cache. Here every sequence has its own length, and with a
`budget` the cache stops growing: after each step every kv head keeps the
newest tokens and those that drew the most attention (the reference serves its
models through `CUDAGraphQuantModel`, modules.py:1589-1691, and leaves the
cache to them). Weights are random, as in `QuantDecoder`.

    model = PagedDecoder(DecoderConfig(...), "cuda", max_batch=8, max_len=4096, budget=1024, recent=128)
    model.calibrate(samples)                # nvfp4: the activations' tensor scales, once
    token = model.prefill(prompts)          # list of 1-D token tensors, one per sequence
    for _ in range(min(n, model.steps_left)):
        token = model.decode_step(token)    # may be captured in a CUDA graph

    model = PagedDecoder(DecoderConfig(...), "cuda", format="int8", cache_dtype=torch.int8, qk_norm=True, pages=2000,
                         max_batch=64, max_len=8192)    # 64 sequences of 8192 tokens would take 8192 pages of 64

A step that a sequence has no rotary row or no slot for raises; the others go
on once that one is taken out (`drop`). Replays of a captured step run without
the host: the program counts them with `count_steps`, which raises for them.
Without that, a sequence past its limit keeps its cache as it is, and its
logits mean nothing.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import torch
import torch.nn.functional as F
from torch import nn

from .decoder import DecoderConfig, _rms_norm, student_t_weight
from .fp4 import Fp4Linear, fp4_quantize
from .int8 import Int8Linear, int8_quantize
from .paged import (PagedKVCache, PagedKVCache8, PagePool, paged_append, paged_decode_attention, paged_evict, paged_release,
                    paged_reserve, qk_norm_rope)


def _prompt_weights(q: torch.Tensor, k: torch.Tensor, lens: Sequence[int], most: int = 1 << 26) -> torch.Tensor:
    """The weight that each prompt token draws from its own prompt: [batch,
    n_kv, tokens], fp32, summed over the prompt's queries and each kv head's query
    heads, as `paged_decode_attention` accumulates it step by step. q [batch,
    tokens, n_heads, D] and k [batch, tokens, n_kv, D] are rotated; lens[b] tokens
    of sequence b count. Scores and softmax are fp32, in blocks of queries of at
    most `most` scores. (4 prompts of 4096 tokens, 32 heads over 8 of 128 columns:
    see the figure at `PagedDecoder.prefill`.)"""
    B, T, H, D = q.shape
    n_kv = k.shape[2]
    q = q.view(B, T, n_kv, H // n_kv, D).transpose(1, 2)                     # a token's query heads side by side
    k = k.permute(0, 2, 3, 1)
    total = torch.zeros(B, n_kv, T, dtype=torch.float32, device=q.device)
    none = total.new_zeros(())
    for b, n in enumerate(lens):
        rows = max(1, most // (H * n))
        for i in range(0, n, rows):
            j = min(n, i + rows)                                              # queries i .. j - 1 see keys 0 .. j - 1
            s = torch.baddbmm(none.expand(n_kv, (j - i) * (H // n_kv), j), q[b, :, i:j].reshape(n_kv, -1, D), k[b, :, :, :j],
                              beta=0, alpha=D ** -0.5, out_dtype=torch.float32)
            late = torch.ones(j - i, j - i, dtype=torch.bool, device=q.device).triu(1)
            s.view(n_kv, j - i, -1, j)[..., i:].masked_fill_(late[:, None], float("-inf"))
            total[b, :, :j] += s.softmax(dim=-1).sum(dim=1)
    return total


class PagedDecoderLayer(nn.Module):
    """One layer's projections (q/k/v and gate/up fused by rows) and norms."""

    def __init__(self, cfg: DecoderConfig, layer_idx: int, format: str, device, qk_norm: bool = False):
        super().__init__()
        H, D = cfg.hidden, cfg.head_dim
        shapes = {"qkv": ((cfg.n_heads + 2 * cfg.n_kv_heads) * D, H), "o": (H, cfg.n_heads * D),
                  "gate_up": (2 * cfg.intermediate, H), "down": (H, cfg.intermediate)}
        for j, (name, shape) in enumerate(shapes.items()):
            w = student_t_weight(shape, seed=cfg.seed * 100003 + layer_idx * 16 + j, device=device)
            setattr(self, name, Int8Linear(int8_quantize(w)) if format == "int8" else Fp4Linear(fp4_quantize(w, format)))
        self.input_norm = nn.Parameter(torch.ones(H, dtype=torch.float32, device=device), requires_grad=False)
        self.post_norm = nn.Parameter(torch.ones(H, dtype=torch.float32, device=device), requires_grad=False)
        for name in ("q_norm", "k_norm"):
            w = nn.Parameter(torch.ones(D, dtype=torch.float32, device=device), requires_grad=False) if qk_norm else None
            self.register_parameter(name, w)

    def projections(self) -> List[nn.Module]:
        return [self.qkv, self.o, self.gate_up, self.down]


class PagedDecoder(nn.Module):
    """See the module documentation. budget: tokens that each sequence's cache
    is cut back to after a step (None: it grows up to max_len); recent: how many of
    them are the newest whatever their weight. With a budget the caches keep
    each slot's accumulated attention weight and position. max_position: the
    rotary tables' rows, tokens that a sequence can have in all; max_len by
    default, and LONG (33 MB of tables for heads of 128) with a budget, under
    which sequences go on beyond max_len.

    format: "nvfp4", "mxfp4" or "int8". cache_dtype: the cache's type, bf16, or int8 or
    float8_e4m3fn (not with a budget: such a cache evicts nothing). qk_norm: norms of
    each query and key head in front of the rotation. pages: pages that the sequences
    share, each taking them as it grows (None: every sequence has its own for max_len
    tokens; not with a budget)."""

    LONG = 65536

    def __init__(self, cfg: DecoderConfig, device, format: str = "nvfp4", max_batch: int = 1, max_len: int = 2048,
                 page_size: int = 64, max_position: Optional[int] = None, budget: Optional[int] = None, recent: int = 0,
                 cache_dtype: torch.dtype = torch.bfloat16, qk_norm: bool = False, pages: Optional[int] = None):
        super().__init__()
        self.cfg, self.device = cfg, torch.device(device)
        self.budget, self.recent = budget, recent
        if budget is not None and not 0 <= recent <= budget < max_len:
            raise ValueError(f"recent <= budget < max_len is needed, got {recent}, {budget}, {max_len}")
        self.packed = pages is not None or cache_dtype != torch.bfloat16
        if self.packed and budget is not None:
            raise ValueError("a budget needs a cache of bf16 and pages of each sequence's own")
        H, D = cfg.hidden, cfg.head_dim
        g = torch.Generator(device=self.device).manual_seed(cfg.seed + 7)
        self.embed = (torch.randn(cfg.vocab, H, generator=g, device=self.device) * 0.02).to(torch.bfloat16)
        self.lm_head = (torch.randn(cfg.vocab, H, generator=g, device=self.device) * 0.02).to(torch.bfloat16)
        self.final_norm = torch.ones(H, dtype=torch.float32, device=self.device)
        self.layers = nn.ModuleList(PagedDecoderLayer(cfg, i, format, self.device, qk_norm) for i in range(cfg.n_layers))
        positions = max_position or (max_len if budget is None else max(max_len, self.LONG))
        inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, D, 2, device=self.device, dtype=torch.float32) / D))
        ang = torch.outer(torch.arange(positions, device=self.device, dtype=torch.float32), inv)
        self.rope_cos, self.rope_sin = ang.cos(), ang.sin()
        self.pages = pages
        if self.packed:
            self._share_pages(max_batch, max_len, page_size, cache_dtype)
        else:
            self.caches = [PagedKVCache.allocate(max_batch, cfg.n_kv_heads, D, max_len, page_size, device=self.device,
                                                 track=budget is not None) for _ in range(cfg.n_layers)]
        self.positions = torch.zeros(max_batch, dtype=torch.int64, device=self.device)   # of the next token
        self._tokens: List[Optional[int]] = [0] * max_batch   # the same as the host counts them; None: dropped

    def _share_pages(self, batch: int, max_len: int, page_size: int, dtype: torch.dtype) -> None:
        """Caches of all layers with one page table and one count of tokens."""
        cfg, per = self.cfg, -(-max_len // page_size)
        table = torch.full((batch, per), -1, dtype=torch.int32, device=self.device)
        self.pool = PagePool.allocate(self.pages or 0, self.device)
        if self.pages is None:
            table.copy_(torch.arange(batch * per, device=self.device).view(batch, per))
        lens = torch.zeros(batch, dtype=torch.int32, device=self.device)
        shape = (batch * per if self.pages is None else self.pages, cfg.n_kv_heads, page_size, cfg.head_dim)
        self.caches = []
        for _ in range(cfg.n_layers):
            k, v = (torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(2))
            if dtype == torch.bfloat16:
                self.caches.append(PagedKVCache(k, v, table, lens))
                continue
            block = 16                                       # tokens that share a scale: 4 bytes to 16 * head_dim
            ks, vs = (torch.ones(*shape[:2], page_size // block, dtype=torch.float32, device=self.device) for _ in range(2))
            self.caches.append(PagedKVCache8(k, v, ks, vs, table, lens))

    def packed_nbytes(self) -> int:
        """Bytes of the projections' weights."""
        return sum(p.weight().nbytes() for layer in self.layers for p in layer.projections())

    @property
    def longest_sequence(self) -> int:
        """Tokens that a sequence can have: rotary rows and, without a budget, slots."""
        rows = self.rope_cos.shape[0]
        return rows if self.budget is not None else min(rows, self.caches[0].capacity)

    @property
    def steps_left(self) -> int:
        """Decode steps until a sequence has no place for its token: no rotary row, no slot or no page."""
        tokens = [n for n in self._tokens if n is not None]
        steps = self.longest_sequence - max(tokens, default=0)
        if self.pages is not None:
            least, most = 0, steps                           # pages are enough for `least` steps
            while least < most:
                mid = (least + most + 1) // 2
                if self._pages_for(n + mid for n in tokens) <= self.pages:
                    least = mid
                else:
                    most = mid - 1
            steps = least
        return steps

    def _pages_for(self, lens) -> int:
        return sum(-(-n // self.caches[0].page_size) for n in lens)

    def count_steps(self, n: int = 1) -> None:
        """Count n decode steps (negative: steps that the program took back);
        raises if fewer are left. `decode_step` does it by itself, except while
        it is captured: a program that replays a captured step counts each replay."""
        tokens = [t for t in self._tokens if t is not None]
        slots = self.longest_sequence - max(tokens, default=0)
        if n <= slots and self.pages is not None and n > 0 and self._pages_for(t + n for t in tokens) > self.pages:
            raise RuntimeError(f"{n} decode steps, but {self.pages} pages hold {self.steps_left} (see pages and drop)")
        if n > slots:
            raise RuntimeError(f"{n} decode steps, but a sequence has {self.longest_sequence - slots} of "
                               f"{self.longest_sequence} tokens (see max_position, max_len and drop)")
        self._tokens = [None if t is None else t + n for t in self._tokens]

    def drop(self, sequence: int) -> None:
        """Take a sequence out of the steps that follow, until the next
        prefill: it no longer counts, its cache is empty, its pages are the
        others' and its logits mean nothing."""
        self._tokens[sequence] = None
        if self.pages is not None:
            keep = torch.full_like(self.caches[0].seq_lens, -1)
            keep[sequence] = 0
            paged_release(self.pool, self.caches[0], keep)
        for cache in self.caches:
            cache.seq_lens[sequence] = -1

    def _evict(self, cache: PagedKVCache) -> None:
        if self.budget is not None:
            paged_evict(cache, self.budget, self.recent)

    def _mlp(self, layer: PagedDecoderLayer, h: torch.Tensor) -> torch.Tensor:
        gate, up = layer.gate_up(_rms_norm(h, layer.post_norm, self.cfg.rms_eps)).chunk(2, dim=-1)
        return h + layer.down(F.silu(gate) * up)

    def _logits(self, h: torch.Tensor) -> torch.Tensor:
        return F.linear(_rms_norm(h, self.final_norm, self.cfg.rms_eps), self.lm_head).float()

    @torch.no_grad()
    def prefill(self, prompts: Sequence[torch.Tensor], return_logits: bool = False) -> torch.Tensor:
        """Run one prompt per sequence (1-D token tensors, of any lengths up to
        max_len; max_batch of them) from position 0 and fill the caches. Returns the greedy
        next tokens [batch], or the logits [batch, vocab]."""
        cfg, D = self.cfg, self.cfg.head_dim
        B, lens = len(prompts), [len(p) for p in prompts]
        most = min(self.caches[0].capacity, self.rope_cos.shape[0])
        if B != self.positions.shape[0] or min(lens) < 1 or max(lens) > most:
            raise ValueError(f"{self.positions.shape[0]} prompts of 1 to {most} tokens are needed")
        if self.pages is not None and self._pages_for(lens) > self.pages:
            raise ValueError(f"the prompts take {self._pages_for(lens)} pages of {self.pages}")
        if self.packed:
            return self._prefill_packed(prompts, lens, return_logits)
        T = max(lens)
        self._tokens = list(lens)
        tokens = torch.zeros(B, T, dtype=torch.long, device=self.device)
        for i, p in enumerate(prompts):
            tokens[i, :lens[i]] = p.to(self.device)
        n_new = torch.tensor(lens, dtype=torch.int32, device=self.device)
        self.positions.zero_()
        h = self.embed[tokens].float()
        cos, sin = self.rope_cos[:T, None], self.rope_sin[:T, None]

        def rope(x):
            x1, x2 = x.float().chunk(2, dim=-1)
            return torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1).to(x.dtype)

        for layer, cache in zip(self.layers, self.caches):
            x = _rms_norm(h, layer.input_norm, cfg.rms_eps)
            qkv, heads = layer.qkv(x), [cfg.n_heads, cfg.n_kv_heads, cfg.n_kv_heads]
            cache.seq_lens.zero_()
            if layer.q_norm is not None:
                where = torch.arange(T, device=self.device).repeat(B)
                qkv = qk_norm_rope(qkv.view(B * T, -1), *heads[:2], layer.q_norm, layer.k_norm, where, self.rope_cos,
                                   self.rope_sin, cfg.rms_eps)
                rq, rk, v = qkv.view(B, T, -1, D).split(heads, dim=2)
                paged_append(rk, v, cache, self.positions, n_new=n_new,
                             scores=_prompt_weights(rq, rk, lens) if self.budget is not None else None)
            else:
                q, k, v = qkv.view(B, T, -1, D).split(heads, dim=2)
                rq, rk = rope(q), rope(k)
                paged_append(k, v, cache, self.positions, self.rope_cos, self.rope_sin, n_new=n_new,
                             scores=_prompt_weights(rq, rk, lens) if self.budget is not None else None)
            cache.seq_lens.copy_(n_new)
            self._evict(cache)
            # padding stands behind a prompt's tokens: causal attention never looks at it
            a = F.scaled_dot_product_attention(rq.transpose(1, 2), rk.transpose(1, 2), v.transpose(1, 2),
                                               is_causal=True, enable_gqa=True)
            h = self._mlp(layer, h + layer.o(a.transpose(1, 2).reshape(B, T, -1)))
        self.positions.copy_(n_new)
        logits = self._logits(h[torch.arange(B, device=self.device), n_new.long() - 1])
        return logits if return_logits else logits.argmax(dim=-1)

    def _prefill_packed(self, prompts: Sequence[torch.Tensor], lens: List[int], return_logits: bool) -> torch.Tensor:
        """Prefill of prompts one behind the other, without padding, into caches
        that share their pages."""
        cfg, D, cache0 = self.cfg, self.cfg.head_dim, self.caches[0]
        self._tokens = list(lens)
        n_new = torch.tensor(lens, dtype=torch.int32, device=self.device)
        if self.pages is not None:
            paged_release(self.pool, cache0, torch.zeros_like(n_new))
        cache0.seq_lens.zero_()
        got = paged_reserve(self.pool, cache0, n_new, sum(lens))
        ends = torch.tensor(lens).cumsum(0)
        h = self.embed[torch.cat([p.to(self.device) for p in prompts])].float()
        n_q, n_kv = cfg.n_heads, cfg.n_kv_heads
        for layer, cache in zip(self.layers, self.caches):
            qkv = layer.qkv(_rms_norm(h, layer.input_norm, cfg.rms_eps))
            args = (qkv, n_q, n_kv, layer.q_norm, layer.k_norm, got.positions, self.rope_cos, self.rope_sin, cfg.rms_eps)
            if isinstance(cache, PagedKVCache8):
                qkv = qk_norm_rope(*args, out=qkv)
            else:
                qkv = qk_norm_rope(*args, out=qkv, cache=cache, slots=got.slots)
            q, k, v = qkv.view(-1, n_q + 2 * n_kv, D).split([n_q, n_kv, n_kv], dim=1)
            if isinstance(cache, PagedKVCache8):
                paged_append(k, v, cache, n_new=got.granted, offsets=got.offsets)
            a = torch.empty_like(q)
            for end, n in zip(ends.tolist(), lens):
                part = [x[end - n:end].transpose(0, 1)[None] for x in (q, k, v)]
                a[end - n:end] = F.scaled_dot_product_attention(*part, is_causal=True, enable_gqa=True)[0].transpose(0, 1)
            h = self._mlp(layer, h + layer.o(a.reshape(-1, n_q * D)))
        cache0.advance(got.granted)                          # of all layers
        self.positions.copy_(n_new)
        logits = self._logits(h[ends.to(self.device) - 1])
        return logits if return_logits else logits.argmax(dim=-1)

    @torch.no_grad()
    def calibrate(self, prompts: Sequence[torch.Tensor]) -> None:
        """Set the projections' input scales (nvfp4; mxfp4 has none) from a
        prefill of sample prompts, each from what it is given behind the
        projections already set ("int8" finds its scales as it goes: nothing to set). They are 1 before: a block whose largest value
        is below 6 * 2^-6 then has a scale below E4M3's normal range, and its values
        up to three bits less. The caches are left as after `prefill`."""
        keep = torch.arange(max(map(len, prompts), default=0)) < torch.tensor([len(p) for p in prompts])[:, None]
        keep = keep.to(self.device)                      # (not the padding)
        hooks = [p.register_forward_pre_hook(lambda proj, args: proj.calibrate(args[0] if self.packed else args[0][keep]))
                 for layer in self.layers for p in layer.projections() if isinstance(p, Fp4Linear)]
        try:
            self.prefill(prompts)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def decode_step(self, tokens: torch.Tensor, return_logits: bool = False) -> torch.Tensor:
        """One token per sequence at its own position. Returns the greedy next
        tokens [batch], or the logits [batch, vocab]. Raises if a sequence has
        no place for its token (`steps_left`)."""
        self.count_steps(1)
        if torch.cuda.is_current_stream_capturing():
            self.count_steps(-1)                         # nothing runs yet
        # which sequences' caches take the token: all but the dropped ones, and those of uncounted replays
        taken = ((self.positions < self.longest_sequence) & (self.caches[0].seq_lens >= 0)).to(torch.int32)
        if self.packed:
            # pages for the tokens; a sequence that gets none (in replays that nobody counts) stays as it is
            taken = paged_reserve(self.pool, self.caches[0], taken, 0).granted
        views = self.caches
        if self.budget is not None and self.layers[0].q_norm is not None:
            # The rotation in front of the attention turns a sequence past its limit away; the attention, which has
            # no tables then, would still give its slots weights: there it takes no part.
            lens = self.caches[0].seq_lens.masked_fill(taken == 0, -1)
            views = [PagedKVCache(c.k_pages, c.v_pages, c.page_table, lens, c.scores, c.slot_pos) for c in self.caches]
        h = self.embed[tokens].float()
        for layer, cache, view in zip(self.layers, self.caches, views):
            qkv = layer.qkv(_rms_norm(h, layer.input_norm, self.cfg.rms_eps))
            rope = (self.rope_cos, self.rope_sin)
            if layer.q_norm is not None:
                qkv = qk_norm_rope(qkv, self.cfg.n_heads, self.cfg.n_kv_heads, layer.q_norm, layer.k_norm, self.positions, *rope,
                                   self.cfg.rms_eps, out=qkv)
                rope = (None, None)
            a = paged_decode_attention(qkv, self.cfg.n_heads, view, self.positions, *rope, accumulate=self.budget is not None)
            if not self.packed:
                cache.advance(taken)
                self._evict(cache)
            h = self._mlp(layer, h + layer.o(a))
        if self.packed:
            self.caches[0].advance(taken)                    # of all layers
        self.positions.add_(1)
        logits = self._logits(h)
        return logits if return_logits else logits.argmax(dim=-1)
