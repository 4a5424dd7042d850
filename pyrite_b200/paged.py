"""Requests of different lengths decoded together, behind a shared prefix, sampled.

:class:`PagedDecoder` is the multi-sequence decoder
(:class:`pyrite_b200.batch.BatchDecoder`) for serving:

* prompts of any lengths; every request stops at its own end, and its row then
  takes no more pages and reads no more keys of its own;
* a prefix (a system prompt, a document) that all requests continue is run and
  stored once, and read once per step for all of them;
* keys and values live in pages handed out on the GPU as requests grow, in
  fp32 (the reference's cache, executor.py:78-140), fp16 or bf16;
* tokens by temperature, top-k, top-p and min-p (sampler.py:17-45) with each
  request's own settings, from random numbers that the caller may give;
  temperature 0 is greedy (sampler.py:12-15).

One step of all requests is one CUDA graph: pyrite_b200.kernels.paged and
pyrite_b200.kernels.sampling around the projections of BatchDecoder.
"""
from __future__ import annotations

import torch

from .batch import BatchDecoder
from .kernels import paged, sampling
from .kernels.cuda import _check


class PagedDecoder(BatchDecoder):
    """Up to ``batch`` requests of one checkpoint over a paged cache.

    ``max_ctx``: the most positions of a request, the prefix included.
    ``n_pages``: pages of the cache (default: enough for every request at
    ``max_ctx`` and a prefix beside them).
    """

    def __init__(self, spec, tensors, device="cuda", max_ctx: int = 512, batch: int = 16, replicate: bool = False,
                 page_size: int = 16, kv_dtype: torch.dtype = torch.float32, n_pages: int | None = None):
        if not 16 <= page_size <= 256 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 256")
        if kv_dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise ValueError("kv_dtype must be float32, float16 or bfloat16")
        self.page_size, self.kv_dtype = page_size, kv_dtype
        self.width = -(-max_ctx // page_size)
        self.n_pages = (batch + 1) * self.width if n_pages is None else n_pages
        if self.n_pages < 1:
            raise ValueError("n_pages must be at least 1")
        super().__init__(spec, tensors, device=device, max_ctx=max_ctx, batch=batch, replicate=replicate)
        if spec.head_dim != paged.HEAD_DIM:
            raise ValueError("the head dimension must be 128")
        d, B = self.dev, batch
        i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=d)  # noqa: E731
        f32 = lambda fill: torch.full((B,), fill, device=d)  # noqa: E731
        self.free_pages = torch.arange(self.n_pages, dtype=torch.int32, device=d)
        self.used = i32(1)
        self.table = torch.full((B, self.width), -1, dtype=torch.int32, device=d)
        self.slots = paged.TokenSlots.empty(B, row_stride=1, device=d)
        self.lens, self.fresh, self.current = i32(B), i32(B), i32(B)
        self.attended = i32(B)  # own tokens that a step's attention reads: none of a request that has ended
        self.prompt_lens, self.limits = i32(B), i32(B)
        self.temperature, self.top_k, self.top_p, self.min_p = f32(0.0), i32(B), f32(1.0), f32(0.0)
        self.uniforms, self.ids, self.probs = f32(0.0), i32(B), f32(0.0)
        self.prefix: list[int] = []
        self.prefix_pages = torch.full((self.width,), -1, dtype=torch.int32, device=d)
        self.workspace: torch.Tensor | None = None
        self._prefix_cached = True  # the one-sequence caches hold the prefix

    def _alloc_cache(self) -> None:
        s = self.spec
        shape = (s.num_hidden_layers, self.n_pages, s.num_key_value_heads, self.page_size, s.head_dim)
        self.pk = torch.zeros(shape, dtype=self.kv_dtype, device=self.dev)
        self.pv = torch.zeros_like(self.pk)
        self.pools = [paged.KVPool(k, v) for k, v in zip(self.pk, self.pv)]

    # ------------------------------------------------------------------ one step of every request
    def _bembed(self, st: int) -> None:
        s = self.spec
        paged.page_tables(self.lens, self.fresh, self.page_size, self.free_pages, self.used, self.table, self.slots)
        torch.mul(self.slots.kv_lens, self.fresh, out=self.attended)
        _check(self.lib.pyrite_cuda_embed_rows(self.embd.ggml_type, self.embd.data.data_ptr(), s.vocab_size,
                                               s.hidden_size, self.current.data_ptr(), 1, None, self.batch,
                                               self.bhid.data_ptr(), s.hidden_size, st), "embed rows")

    def _battend(self, li: int, ly, st: int) -> None:
        s, n = self.spec, len(self.prefix)
        paged.append_kv(self.bqkv, self.pools[li], self.slots.slots, self.slots.positions, self.rope,
                        s.num_attention_heads, q_norm=ly.q_norm, k_norm=ly.k_norm, eps=float(s.rms_norm_eps), first=n,
                        q_out=self.bq)
        paged.attention(self.bq, self.pools[li], self.table, self.attended, prefix_pages=self.prefix_pages,
                        prefix_len=n, out=self.batt, workspace=self.workspace)

    def _bnext(self, st: int) -> None:
        sampling.sample_rows(self.blogits, self.uniforms, self.temperature, top_k=self.top_k, top_p=self.top_p,
                             min_p=self.min_p, out=self.ids, probs=self.probs)
        _check(self.lib.pyrite_cuda_commit_tokens(
            self.ids.data_ptr(), self.batch, self.btokens.data_ptr(), self.max_ctx, self.lens.data_ptr(),
            self.fresh.data_ptr(), self.current.data_ptr(), self.prompt_lens.data_ptr(), self.limits.data_ptr(), st),
            "commit tokens")

    def bcapture(self) -> None:
        s = self.spec
        self.workspace = paged.attention_workspace(self.batch, s.num_attention_heads, s.num_key_value_heads,
                                                   len(self.prefix), self.kv_dtype, self.dev)
        state = (self.lens, self.fresh, self.current, self.btokens, self.table, self.used)
        saved = [t.clone() for t in state]
        stream = torch.cuda.Stream(device=self.dev)
        torch.cuda.synchronize(self.dev)
        with torch.cuda.device(self.dev), torch.cuda.stream(stream):
            self._bstep(stream.cuda_stream)  # warm: kernel attributes are set before capture
            torch.cuda.synchronize(self.dev)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                self._bstep(stream.cuda_stream)
        torch.cuda.synchronize(self.dev)
        for t, s0 in zip(state, saved):
            t.copy_(s0)
        self.bgraph = g

    # ------------------------------------------------------------------ public
    def reset(self, prompt: list[int]) -> None:
        super().reset(prompt)
        self._prefix_cached = False

    def breset(self, prompts: list[list[int]]) -> None:
        raise NotImplementedError("requests of a paged decoder start with preset")

    def bgenerate(self, prompts: list[list[int]], max_new_tokens: int) -> list[list[int]]:
        """Greedy continuations, as BatchDecoder.bgenerate (here of any lengths, behind the prefix)."""
        if max_new_tokens == 0:
            return [list(p) for p in prompts]
        return self.pgenerate(prompts, max_new_tokens)

    def set_prefix(self, tokens: list[int], prefill_block: int = 64) -> None:
        """Run ``tokens`` once; every request of the following calls continues them ([]: no prefix)."""
        tokens = [int(t) for t in tokens]
        if any(not 0 <= t < self.spec.vocab_size for t in tokens):
            raise ValueError("prefix token ids must lie inside the vocabulary")
        if len(tokens) + 2 > self.max_ctx:
            raise ValueError("the prefix leaves no room in the context")
        n = len(tokens)
        if -(-n // self.page_size) > self.n_pages:
            raise ValueError("the prefix does not fit the pages")
        # until all of it is done there is no prefix; the captured step has the old one's length in it
        graph, self.bgraph = (self.bgraph if n == len(self.prefix) else None), None
        self.prefix = []
        self.used.zero_()
        if n:
            self.prefill(tokens + tokens[-1:], max(1, prefill_block))  # positions 0 .. n - 1 into the one-sequence caches
            one = lambda v: torch.tensor([v], dtype=torch.int32, device=self.dev)  # noqa: E731
            slots = paged.TokenSlots.empty(1, capacity=n, device=self.dev)
            paged.page_tables(one(0), one(n), self.page_size, self.free_pages, self.used, self.prefix_pages[None],
                              slots)
            for li, pool in enumerate(self.pools):
                paged.store_kv(self.kcache[li][:n], self.vcache[li][:n], pool, slots.slots)
        torch.cuda.synchronize(self.dev)
        self.check_status()
        self.prefix, self.bgraph, self._prefix_cached = tokens, graph, True

    def _setting(self, t: torch.Tensor, value, count: int, name: str) -> None:
        values = list(value) if isinstance(value, (list, tuple)) else [value] * count
        if len(values) != count:
            raise ValueError(f"{name}: one value, or one per prompt")
        t[:count] = torch.tensor(values, dtype=t.dtype, device=self.dev)

    def preset(self, prompts: list[list[int]], max_new_tokens: int | list[int]) -> None:
        """Up to ``batch`` prompts of any lengths (without the prefix); rows past the last prompt stay empty."""
        n, P = len(prompts), len(self.prefix)
        if not 1 <= n <= self.batch:
            raise ValueError(f"1 to {self.batch} prompts expected, got {n}")
        new = list(max_new_tokens) if isinstance(max_new_tokens, (list, tuple)) else [max_new_tokens] * n
        if len(new) != n or any(m < 1 for m in new):
            raise ValueError("max_new_tokens must be at least 1, one value or one per prompt")
        if any(not p for p in prompts) or any(P + len(p) + m > self.max_ctx for p, m in zip(prompts, new)):
            raise ValueError("prompts must be non-empty and fit the context with the prefix and the new tokens")
        if any(not 0 <= t < self.spec.vocab_size for p in prompts for t in p):
            raise ValueError("prompt token ids must lie inside the vocabulary")
        ps, held = self.page_size, -(-P // self.page_size)
        # the last token of a request is never run, so it takes no slot
        if held + sum(-(-(len(p) + m - 1) // ps) for p, m in zip(prompts, new)) > self.n_pages:
            raise ValueError("the requests do not fit the pages")
        B, mc = self.batch, self.max_ctx
        tok = torch.zeros(B, mc, dtype=torch.int32)
        rows = torch.zeros(5, B, dtype=torch.int32)  # lens, fresh, current, prompt_lens, limits
        for j, (p, m) in enumerate(zip(prompts, new)):
            tok[j, :len(p)] = torch.tensor(p, dtype=torch.int32)
            rows[1, j], rows[2, j], rows[3, j], rows[4, j] = 1, p[0], len(p), len(p) + m
        self.btokens.copy_(tok)
        for t, r in zip((self.lens, self.fresh, self.current, self.prompt_lens, self.limits), rows):
            t.copy_(r)
        self.table.fill_(-1)
        self.used.fill_(held)

    def _prefill_prompts(self, prompts: list[list[int]], block: int) -> None:
        """Every prompt but its last token through multi-column products, one
        prompt after the other behind the prefix (still in the one-sequence
        caches), its keys and values copied into its slots."""
        P, counts = len(self.prefix), [len(p) - 1 for p in prompts]
        if sum(counts) == 0:
            return
        d = self.dev
        if P and not self._prefix_cached:  # another prompt has run through the one-sequence caches
            self.prefill(self.prefix + self.prefix[-1:], block)
            self._prefix_cached = True
        new = torch.zeros(self.batch, dtype=torch.int32)
        new[:len(prompts)] = torch.tensor(counts, dtype=torch.int32)
        slots = paged.TokenSlots.empty(self.batch, capacity=sum(counts), device=d)
        paged.page_tables(self.lens, new.to(d), self.page_size, self.free_pages, self.used, self.table, slots)
        at = 0
        for j, (p, n) in enumerate(zip(prompts, counts)):
            if n == 0:
                continue
            self.tokens[P:P + n] = torch.tensor(p[:n], dtype=torch.int32, device=d)
            self._prefill_rows(P, P + n, block)
            for li, pool in enumerate(self.pools):
                paged.store_kv(self.kcache[li][P:P + n], self.vcache[li][P:P + n], pool, slots.slots[at:at + n])
            self.current[j] = p[n]
            at += n
        self.lens.copy_(slots.kv_lens)

    def pgenerate(self, prompts: list[list[int]], max_new_tokens: int | list[int], temperature=0.0, top_k=0,
                  top_p=1.0, min_p=0.0, uniforms: torch.Tensor | None = None, seed: int = 0,
                  prefill_block: int = 0) -> list[list[int]]:
        """Continuations of all prompts, each behind the prefix of :meth:`set_prefix`.

        Settings: one value or one per prompt.  ``uniforms``: random numbers
        in [0, 1), (prompts, context) float32, entry (j, t) for the token at
        position t of request j after the prefix; drawn from ``seed`` when
        omitted.  ``prefill_block`` > 0 (dense checkpoints): prompts through
        blocks of that many positions, else one position per step.  Returns
        each prompt with its new tokens (the prefix left out).  Raises
        RuntimeError, naming the requests, where a request met logits of
        nothing but -inf and NaN: it then has no next token."""
        n, d = len(prompts), self.dev
        self.preset(prompts, max_new_tokens)
        for t, v, name in ((self.temperature, temperature, "temperature"), (self.top_k, top_k, "top_k"),
                           (self.top_p, top_p, "top_p"), (self.min_p, min_p, "min_p")):
            self._setting(t, v, n, name)
        if uniforms is None:
            uniforms = torch.rand(n, self.max_ctx, generator=torch.Generator().manual_seed(seed))
        if uniforms.dim() != 2 or uniforms.shape[0] != n or uniforms.shape[1] < int(self.limits.max()):
            raise ValueError("uniforms must hold one random number per prompt and position")
        limits = self.limits[:n].tolist()
        if self.bgraph is None:
            self.bcapture()
        if prefill_block > 0 and not self.moe:
            self._prefill_prompts(prompts, prefill_block)
        first = self.lens[:n].tolist()
        steps = max(m - 1 - f for m, f in zip(limits, first))
        # step i samples the token at position first + i + 1 of each request
        at = torch.tensor(first)[:, None] + 1 + torch.arange(steps)
        draws = uniforms.float().cpu().gather(1, at.clamp(max=uniforms.shape[1] - 1)).t().contiguous().to(d)
        for i in range(steps):
            self.uniforms[:n].copy_(draws[i])
            self.bgraph.replay()
        torch.cuda.synchronize(d)
        self.check_status()
        tokens = self.btokens.cpu()
        outs = [[int(t) for t in tokens[j, :limits[j]]] for j in range(n)]
        stuck = [j for j, out in enumerate(outs) if -1 in out]
        if stuck:
            raise RuntimeError(f"requests {stuck} have no next token: all of their logits were -inf or NaN")
        return outs
