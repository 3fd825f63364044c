"""SmolLM2 forward with the attention path and its callers on the B200 kernels.

The reference's layer (smollm.py:168-253) projects q, k and v, rotates q and k
(apply_rope), grows the layer's (k, v) cache with torch.cat, expands GQA heads
with repeat_interleave and then runs attention on the CPU or through
run_batch. Here the same layer math runs as:

  * one fused QKV projection (wq, wk, wv stacked: a single cuBLAS GEMM);
  * b2a_rope_append: rotation of q and k and an in-place append of k and v
    into a device-resident KVCache, in one launch, heads never expanded;
  * b2a_prefill (T > 1, causal from each sequence's cache position) or
    b2a_decode (T = 1) reading the cache directly;
  * output projection, RMSNorms and the SwiGLU MLP in torch, as in the
    reference.

Prompts of different lengths run packed instead of padded (prefill_packed,
decode_packed, generate): b2a_rope_append_paged writes k and v to the pages of
each sequence (bf16 or 8-bit), b2a_prefill_varlen and b2a_decode_paged attend,
b2a_penalize and b2a_sample choose the tokens. Behind a shared prefix, whose
pages all sequences name, prompts attend the cached keys that b2a_gather_paged
reads back, and single tokens go through b2a_decode_paged_shared.

Sequence positions stay on the device (KVCache), so a decode step issues no
host synchronisation. Weights use the reference's HF key names
(smollm.py:84-93, :256-265). The model may run in fp32 (the reference's NPU
configuration) or bf16; attention always takes bf16 Q/K/V.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as F

from . import api
from .kvcache import KVCache, PagedKVCache, PagedSequences
from .profiler import profile


@dataclass
class SmolLMConfig:
    """Architecture hyper-parameters (the fields of smollm.py:23-34)."""

    dim: int = 576
    n_layers: int = 30
    n_heads: int = 9
    n_kv_heads: int = 3
    head_dim: int = 64
    ffn_dim: int = 1536
    vocab: int = 49152
    max_pos: int = 8192
    rope_theta: float = 100000.0
    rms_eps: float = 1e-5


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """RMSNorm computed in fp32, returned in x's dtype (smollm.py:37-42)."""
    xf = x.float()
    return ((xf * xf.pow(2).mean(-1, keepdim=True).add(eps).rsqrt()) * w.float()).to(x.dtype)


def rope_tables(head_dim: int, max_pos: int, theta: float, dtype, device):
    """Rotary cos/sin [max_pos, head_dim] as build_rope_cache (smollm.py:45-50):
    fp32 angles, halves duplicated, cast to the model dtype."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim))
    ang = torch.outer(torch.arange(max_pos, dtype=torch.float32, device=device), inv)
    ang = torch.cat([ang, ang], dim=-1)
    return ang.cos().to(dtype).contiguous(), ang.sin().to(dtype).contiguous()


class SmolLMB200:
    """Decoder stack over a KVCache; forward(ids, cache) -> logits."""

    def __init__(self, sd: dict, cfg: SmolLMConfig, device: torch.device, dtype: Optional[torch.dtype] = None,
                 fuse_wo: bool = True):
        """fuse_wo: single-token steps run the output projection and residual
        add inside the decode combine kernel (b2a_decode_proj) instead of a
        separate GEMM."""
        dtype = dtype or sd["model.embed_tokens.weight"].dtype
        self.fuse_wo = fuse_wo
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("the model runs in float32 or bfloat16")
        self.cfg, self.device, self.dtype = cfg, device, dtype

        def w(key):
            return sd[key].to(device=device, dtype=dtype).contiguous()

        self.embed = w("model.embed_tokens.weight")
        self.final_norm = w("model.norm.weight")
        self.layers = []
        for i in range(cfg.n_layers):
            p = f"model.layers.{i}."
            self.layers.append({
                "wqkv": torch.cat([w(p + "self_attn.q_proj.weight"), w(p + "self_attn.k_proj.weight"),
                                   w(p + "self_attn.v_proj.weight")], dim=0).contiguous(),
                "wo": w(p + "self_attn.o_proj.weight"),
                "w_gate": w(p + "mlp.gate_proj.weight"),
                "w_up": w(p + "mlp.up_proj.weight"),
                "w_down": w(p + "mlp.down_proj.weight"),
                "ln1": w(p + "input_layernorm.weight"),
                "ln2": w(p + "post_attention_layernorm.weight"),
            })
        self.cos, self.sin = rope_tables(cfg.head_dim, cfg.max_pos, cfg.rope_theta, dtype, device)
        self._ws = None

    def new_cache(self, batch: int, max_len: int) -> KVCache:
        if max_len > self.cfg.max_pos:
            raise ValueError(f"max_len {max_len} exceeds the rotary table length {self.cfg.max_pos}")
        return KVCache(self.cfg.n_layers, batch, self.cfg.n_kv_heads, max_len, self.cfg.head_dim, self.device)

    def _workspace(self, B: int, Lmax: int) -> torch.Tensor:
        c = self.cfg
        need = api.decode_workspace_bytes(B, c.n_heads, c.n_kv_heads, c.head_dim, Lmax)
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        return self._ws

    def _attention(self, lw: dict, h: torch.Tensor, cache: KVCache, i: int, x: torch.Tensor):
        """Attention of layer i; returns the new residual stream (x plus the
        output projection of the attention)."""
        c = self.cfg
        B, T, _ = h.shape
        Hq, Hkv, Dh = c.n_heads, c.n_kv_heads, c.head_dim
        with profile("qkv"):
            qkv = F.linear(h, lw["wqkv"])                                # [B, T, (Hq + 2 Hkv) Dh]
        q = qkv[..., :Hq * Dh].view(B, T, Hq, Dh)
        k = qkv[..., Hq * Dh:(Hq + Hkv) * Dh].view(B, T, Hkv, Dh)
        v = qkv[..., (Hq + Hkv) * Dh:].view(B, T, Hkv, Dh)
        k_cache, v_cache = cache.layer(i)
        with profile("rope"):
            q_rot = api.rope_append(q, k, v, self.cos, self.sin, k_cache, v_cache,
                                    start_pos_per_batch=cache.start, seqlens_out=cache.end)
        if T == 1:
            if self.fuse_wo and x.is_contiguous():
                # Attention, output projection and residual add in one decode
                # (the combine kernel adds o @ wo.T into x in place).
                with profile("attn"):
                    api.decode_proj(q_rot[:, :, 0], k_cache, v_cache, cache.end, lw["wo"], x.view(B, -1),
                                    workspace=self._workspace(B, cache.max_len))
                return x
            with profile("attn"):
                o = api.decode(q_rot[:, :, 0], k_cache, v_cache, cache.end, out_dtype=h.dtype,
                               workspace=self._workspace(B, cache.max_len))
            with profile("wo"):
                return x + F.linear(o.reshape(B, 1, Hq * Dh), lw["wo"])
        # The kernel writes O straight into the [B, T, Hq * Dh] layout the
        # output projection reads (a strided [B, Hq, T, Dh] view of it).
        o = torch.empty((B, T, Hq, Dh), dtype=h.dtype, device=h.device)
        with profile("attn"):
            api.prefill(q_rot, k_cache, v_cache, start_pos_per_batch=cache.start, scale=1.0 / math.sqrt(Dh),
                        causal=True, out_dtype=h.dtype, out=o.transpose(1, 2))
        with profile("wo"):
            return x + F.linear(o.view(B, T, Hq * Dh), lw["wo"])

    @torch.no_grad()
    def capture_decode(self, cache: KVCache, warmup: int = 2):
        """A CUDA graph of one single-token step over `cache` (every layer's
        norm, projections, rope_append, decode attention and MLP: ~12
        launches per layer replayed as one). Returns step(ids [B, 1]) ->
        logits [B, 1, vocab] (a buffer the next replay overwrites). Warm-up and
        capture run real steps; the cache's positions are restored afterwards,
        so the rows they wrote (at most warmup + 1 past each sequence's
        length, which must fit in max_len) are overwritten by the next tokens
        and never read.
        """
        B = cache.batch
        ids_buf = torch.zeros((B, 1), dtype=torch.long, device=self.device)
        self._workspace(B, cache.max_len)  # allocate outside the capture
        saved = cache._pos.clone()
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            for _ in range(warmup):
                self.forward(ids_buf, cache)
        torch.cuda.current_stream(self.device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = self.forward(ids_buf, cache)
        cache._pos.copy_(saved)

        def step(ids: torch.Tensor) -> torch.Tensor:
            ids_buf.copy_(ids)
            graph.replay()
            return out

        step.graph = graph
        return step

    @torch.no_grad()
    def capture_prefill(self, cache: KVCache, T: int, warmup: int = 2):
        """A CUDA graph of one T-token prefill step over `cache` (every layer's
        norms, fused QKV GEMM, rope_append, prefill attention, output
        projection and MLP replayed as one launch), the prefill counterpart of
        capture_decode. Returns step(ids [B, T]) -> logits [B, T, vocab] (a
        buffer the next replay overwrites); each replay appends at the
        cache's current positions and advances them, like forward. Warm-up and
        capture run real steps and the positions are restored afterwards, so
        the rows they wrote are overwritten by the next replay."""
        B = cache.batch
        ids_buf = torch.zeros((B, T), dtype=torch.long, device=self.device)
        saved = cache._pos.clone()
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            for _ in range(warmup):
                cache._pos.copy_(saved)
                self.forward(ids_buf, cache)
        torch.cuda.current_stream(self.device).wait_stream(side)
        cache._pos.copy_(saved)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = self.forward(ids_buf, cache)
        cache._pos.copy_(saved)

        def step(ids: torch.Tensor) -> torch.Tensor:
            ids_buf.copy_(ids)
            graph.replay()
            return out

        step.graph = graph
        return step

    @torch.no_grad()
    def forward(self, ids: torch.Tensor, cache: KVCache) -> torch.Tensor:
        """Logits [B, T, vocab] for tokens ids [B, T] placed after each
        sequence's cached prefix; appends them to the cache."""
        c = self.cfg
        if ids.dim() != 2 or ids.shape[0] != cache.batch:
            raise ValueError("ids must be [B, T] with B = cache.batch")
        x = self.embed[ids.to(self.device)]
        # Op names follow the reference forward's profile() blocks
        # (smollm.py:179-251), with "attn" for its attn_npu / attn_cpu.
        for i, lw in enumerate(self.layers):
            with profile("rms1"):
                h = rms_norm(x, lw["ln1"], c.rms_eps)
            x = self._attention(lw, h, cache, i, x)
            with profile("rms2"):
                h = rms_norm(x, lw["ln2"], c.rms_eps)
            with profile("gate_up"):
                gu = F.silu(F.linear(h, lw["w_gate"])) * F.linear(h, lw["w_up"])
            with profile("w_down"):
                x = x + F.linear(gu, lw["w_down"])
        cache.advance()
        x = rms_norm(x, self.final_norm, c.rms_eps)
        return F.linear(x, self.embed)

    # ------------------------------------------------------------ sequences of different lengths
    def new_paged_cache(self, n_pages: int, page: int = 64, dtype: torch.dtype = torch.bfloat16) -> PagedKVCache:
        """dtype torch.float8_e4m3fn: an 8-bit cache, about half the memory and traffic."""
        c = self.cfg
        return PagedKVCache(c.n_layers, n_pages, c.n_kv_heads, page, c.head_dim, self.device, dtype)

    def _attention_packed(self, lw: dict, h: torch.Tensor, seqs: PagedSequences, i: int,
                          cu_seqlens: Optional[torch.Tensor], cu_keys: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of layer i before the output projection, [N, Hq * Dh]: of
        packed prompts with offsets cu_seqlens (behind a shared prefix, cu_keys
        those of their keys with it), or (None) of one token per sequence
        against its cached keys."""
        c = self.cfg
        Hq, Hkv, Dh = c.n_heads, c.n_kv_heads, c.head_dim
        N = h.shape[0]
        with profile("qkv"):
            qkv = F.linear(h, lw["wqkv"])
        q = qkv[:, :Hq * Dh].view(N, Hq, Dh)
        k = qkv[:, Hq * Dh:(Hq + Hkv) * Dh].view(N, Hkv, Dh)
        v = qkv[:, (Hq + Hkv) * Dh:].view(N, Hkv, Dh)
        k_pages, v_pages = seqs.cache.layer(i)
        scales = seqs.cache.scales(i)
        prompts = cu_seqlens is not None
        behind = prompts and seqs.prefix_tokens > 0
        with profile("rope"):
            rot = api.rope_append_paged(q, k, v, self.cos, self.sin, k_pages, v_pages, seqs.block_table,
                                        cu_seqlens if prompts else seqs.one_each, start_pos_per_batch=seqs.start,
                                        seqlens_out=seqs.end, return_kv=prompts and not behind, **scales)
        with profile("attn"):
            if behind:
                # The prefix's keys and the prompt's own, both as the cache holds them.
                kv = api.gather_paged(k_pages, v_pages, seqs.block_table, cu_keys, N + seqs.batch * seqs.prefix_tokens,
                                      **scales)
                o = api.prefill_varlen(rot, *kv, cu_seqlens, cu_keys, out_dtype=h.dtype)
            elif prompts:
                o = api.prefill_varlen(*rot, cu_seqlens, out_dtype=h.dtype)
            elif seqs.prefix_tokens and not scales:
                o = api.decode_paged_shared(rot, k_pages, v_pages, seqs.block_table, seqs.end, seqs.prefix_lens,
                                            out_dtype=h.dtype)
            else:
                o = api.decode_paged(rot, k_pages, v_pages, seqs.block_table, seqs.end, out_dtype=h.dtype, **scales)
        return o.view(N, Hq * Dh)

    def _forward_packed(self, ids: torch.Tensor, seqs: PagedSequences,
                        cu_seqlens: Optional[torch.Tensor]) -> torch.Tensor:
        """The final norm's output for packed tokens ids [N]; advances seqs."""
        if seqs.released:
            raise ValueError("the sequences are released: their pages may have other owners")
        c = self.cfg
        x = self.embed[ids]
        cu_keys = None
        if cu_seqlens is not None and seqs.prefix_tokens:
            cu_keys = cu_seqlens + seqs.prefix_tokens * seqs.one_each
        for i, lw in enumerate(self.layers):
            with profile("rms1"):
                h = rms_norm(x, lw["ln1"], c.rms_eps)
            o = self._attention_packed(lw, h, seqs, i, cu_seqlens, cu_keys)
            with profile("wo"):
                x = x + F.linear(o, lw["wo"])
            with profile("rms2"):
                h = rms_norm(x, lw["ln2"], c.rms_eps)
            with profile("gate_up"):
                gu = F.silu(F.linear(h, lw["w_gate"])) * F.linear(h, lw["w_up"])
            with profile("w_down"):
                x = x + F.linear(gu, lw["w_down"])
        seqs.advance()
        return rms_norm(x, self.final_norm, c.rms_eps)

    @torch.no_grad()
    def prefill_packed(self, ids: torch.Tensor, cu_seqlens: torch.Tensor, seqs: PagedSequences) -> torch.Tensor:
        """Logits [B, vocab] of each prompt's last token, for prompts packed in
        ids [N] (sequence b: ids[cu_seqlens[b] : cu_seqlens[b + 1]], none empty)
        into the new, empty sequences `seqs` (behind their shared prefix, if they
        have one: its tokens are in the cache already). Of offsets that are not a stretch
        of ids the logits mean nothing; api.device_error() reports them."""
        if ids.dim() != 1 or cu_seqlens.numel() != seqs.batch + 1:
            raise ValueError("ids must be [N] and cu_seqlens [B + 1] with B = seqs.batch")
        x = self._forward_packed(ids.to(self.device), seqs, cu_seqlens)
        last = (cu_seqlens[1:] - 1).long().clamp(0, x.shape[0] - 1)  # an index past the end would fault
        return F.linear(x[last], self.embed)

    @torch.no_grad()
    def decode_packed(self, ids: torch.Tensor, seqs: PagedSequences) -> torch.Tensor:
        """Logits [B, vocab] after one more token ids [B], from 0 on, of every sequence. A
        sequence whose pages are full keeps its keys and its logits mean
        nothing; api.device_error() reports it."""
        if ids.dim() != 1 or ids.numel() != seqs.batch:
            raise ValueError("ids must be [B] with B = seqs.batch")
        return F.linear(self._forward_packed(ids.to(self.device), seqs, None), self.embed)

    @torch.no_grad()
    def generate(self, prompts, max_new_tokens: int, *, cache: Optional[PagedKVCache] = None, page: int = 64,
                 temperature=0.0, top_k=0, top_p=1.0, min_p=0.0,
                 generator: Optional[torch.Generator] = None, prefix=None, repetition_penalty=1.0,
                 frequency_penalty=0.0, presence_penalty=0.0, logit_bias: Optional[torch.Tensor] = None,
                 allowed: Optional[torch.Tensor] = None) -> torch.Tensor:
        """max_new_tokens tokens after each prompt (a list of token lists, of
        any lengths from 1), int64 [B, max_new_tokens] on the device. The
        settings are those of api.sample; temperature 0 is greedy. A prompt
        whose logits hold no usable one gives -1 there and in the rest of its
        row. Nothing synchronises with the host in between.

        prefix: tokens ahead of every prompt (a system prompt), run and stored
        once: their whole pages are shared. Behind them prompts attend keys and
        values as the cache holds them, their own too (with an 8-bit cache
        quantised ones, where prompts without a prefix attend theirs before that),
        and single tokens as api.decode_paged_shared does by default (bf16: P
        rounded to bf16 over the prefix where it is shared) or api.decode_paged
        (8-bit: the prefix read once for every sequence).

        The penalties, logit_bias (bias) and allowed are those of api.penalize,
        over the prefix, the prompt and what was generated; one allowed for all
        steps (a grammar, whose mask follows the tokens, calls api.penalize between
        prefill_packed or decode_packed and api.sample)."""
        lens = [len(p) for p in prompts]
        if not lens or min(lens) < 1 or max_new_tokens < 1:
            raise ValueError("every prompt needs a token and max_new_tokens must be positive")
        flat = [int(t) for p in prompts for t in p]
        prefix = [] if prefix is None else [int(t) for t in prefix]
        if min(flat + prefix) < 0 or max(flat + prefix) >= self.embed.shape[0]:
            raise ValueError(f"prompt tokens must lie in the vocabulary, 0 to {self.embed.shape[0] - 1}")
        room = [n + max_new_tokens - 1 for n in lens]  # the last token is not fed back
        if max(room) + len(prefix) > self.cfg.max_pos:
            raise ValueError(f"{max(room) + len(prefix)} positions exceed the rotary table length {self.cfg.max_pos}")
        page = page if cache is None else cache.page
        shared = len(prefix) // page * page
        prompts = [prefix[shared:] + [int(t) for t in p] for p in prompts]
        lens, room = [len(p) for p in prompts], [r + len(prefix) - shared for r in room]
        if cache is None:
            cache = self.new_paged_cache(shared // page + sum(-(-r // page) for r in room), page)
        head = cache.reserve([shared]) if shared else None
        seqs = None
        try:
            seqs = cache.reserve(room, prefix=head)
            cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(self.device)
            ids = torch.tensor([t for p in prompts for t in p], dtype=torch.long, device=self.device)
            greedy = not isinstance(temperature, torch.Tensor) and temperature <= 0
            out = torch.empty((max_new_tokens, len(lens)), dtype=torch.long, device=self.device)
            adjust = self._penalties([prefix[:shared] + p for p in prompts], max_new_tokens, repetition_penalty,
                                     frequency_penalty, presence_penalty, logit_bias, allowed)
            if shared:
                self.prefill_packed(torch.tensor(prefix[:shared], dtype=torch.long, device=self.device),
                                    torch.tensor([0, shared], dtype=torch.int32, device=self.device), head)
            logits = self.prefill_packed(ids, cu, seqs)
            for step in range(max_new_tokens):
                if adjust is not None:
                    logits = adjust(logits, out[step - 1] if step else None)
                noise = None if greedy else torch.empty(logits.shape, dtype=torch.float32,
                                                        device=self.device).exponential_(generator=generator)
                with profile("sample"):
                    api.sample(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                               out=out[step])
                if step > 0:  # once -1, always -1
                    torch.where(out[step - 1] < 0, out[step - 1], out[step], out=out[step])
                if step + 1 < max_new_tokens:
                    logits = self.decode_packed(out[step].clamp(min=0), seqs)
        finally:
            if seqs is not None:
                seqs.release()
            if head is not None:
                head.release()
        return out.T.contiguous()

    def _penalties(self, prompts: list, new_tokens: int, repetition, frequency, presence, bias, allowed):
        """adjust(logits, the tokens of the step before) -> logits for generate, or None if nothing applies."""
        def off(value, neutral):
            return not isinstance(value, torch.Tensor) and value == neutral

        if off(repetition, 1.0) and off(frequency, 0.0) and off(presence, 0.0):
            if bias is None and allowed is None:
                return None
            return lambda logits, last: api.penalize(logits, bias=bias, allowed=allowed, out=logits)
        lens = [len(p) for p in prompts]
        history = torch.full((len(lens), max(lens) + new_tokens), -1, dtype=torch.long)
        for b, p in enumerate(prompts):
            history[b, :len(p)] = torch.tensor(p, dtype=torch.long)
        history = history.to(self.device)
        prompt_lengths = torch.tensor(lens, dtype=torch.int32, device=self.device)
        lengths = prompt_lengths.clone()

        def adjust(logits, last):
            if last is not None:
                history.scatter_(1, lengths[:, None].long(), last[:, None])
                lengths.add_(1)
            with profile("penalize"):
                return api.penalize(logits, history, lengths, prompt_lengths=prompt_lengths, repetition=repetition,
                                    frequency=frequency, presence=presence, bias=bias, allowed=allowed, out=logits)

        return adjust
