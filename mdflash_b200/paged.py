"""A paged K/V cache shared by many requests, and the decoding loop that runs on it.

The verify path keeps one contiguous cache per request (cache.py), as the reference does
(ddtree.py:387).  A server that holds many requests of changing length keeps their K/V in
pages instead: ``PagedKVCache`` is the page pools of every layer, the requests' block tables
and the free stack, all on the device, and ``PagedKVCache.step`` moves every request from its
length to its next one in one launch (K.page_tables): a prompt's chunk enters, a decoded token
is added, rejected drafts roll back, an ended request gives its pages back.

``paged_generate`` answers a list of prompts with it: prompts enter in chunks beside the
requests that already decode, one forward per step for all of them
(Qwen3VerifyRunner.forward_paged), and K.sample draws every finished row's token.
"""
from __future__ import annotations

import torch

from . import _lib
from . import kernels as K


class PagedKVCache:
    """Page pools of ``num_layers`` layers, K and V each bf16 [n_pages, kv_heads, page_size,
    head_dim], and the tables of ``max_requests`` places of at most ``max_pages`` pages."""

    def __init__(self, num_layers: int, n_pages: int, kv_heads: int, head_dim: int,
                 max_requests: int, max_pages: int, page_size: int = 16,
                 device: torch.device | str = "cuda"):
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 1024")
        self.device = torch.device(device)
        self.page_size, self.max_pages, self.n_pages = page_size, max_pages, n_pages
        shape = (n_pages, kv_heads, page_size, head_dim)
        bf16 = dict(dtype=torch.bfloat16, device=self.device)
        self.k_pages = [torch.empty(shape, **bf16) for _ in range(num_layers)]
        self.v_pages = [torch.empty(shape, **bf16) for _ in range(num_layers)]
        i32 = dict(dtype=torch.int32, device=self.device)
        self.block_table = torch.zeros((max_requests, max_pages), **i32)
        self.lens = torch.zeros(max_requests, **i32)
        # taken from the top: page 0 first
        self.free_pages = torch.arange(n_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), n_pages, **i32)
        self.status = torch.zeros(1, **i32)

    @property
    def max_requests(self) -> int:
        return self.lens.numel()

    def step(self, new_lens: torch.Tensor, max_tokens: int) -> K.PageStep:
        """Moves every place from its length to ``new_lens`` (i32 [max_requests], device), with
        at most ``max_tokens`` new tokens in all.  The returned step's tensors are its own but
        kv_lens and free_count, which are the cache's.  A step that does not fit changes
        nothing and sets the status word (check)."""
        out = K.PageStep.allocate(self.device, self.max_requests, max_tokens)
        out.kv_lens, out.free_count = self.lens, self.free_count
        return K.page_tables(self.lens, new_lens, self.block_table, self.free_pages,
                             self.free_count, self.page_size, max_tokens, out=out,
                             status=self.status)

    def check(self) -> None:
        """Raises DDTreeError when a step or an attention launch reported an error (syncs)."""
        K.check_status(self.status, "paged cache")


@torch.inference_mode()
def paged_generate(runner, prompts: list[torch.Tensor], max_new_tokens: int,
                   temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
                   stop_token_ids=None, chunk_tokens: int = 2048, page_size: int = 16,
                   n_pages: int | None = None,
                   generator: torch.Generator | None = None) -> list[torch.Tensor]:
    """Answers every prompt (i64 [n_i]) with up to max_new_tokens tokens drawn by K.sample and
    returns the new tokens (CPU) per prompt.  runner: a Qwen3VerifyRunner.  A step takes one
    token of every decoding request and fills up to chunk_tokens with the next chunks of the
    prompts; the uniforms come from ``generator`` (torch's default one without it), one per
    drawn token.  n_pages: the pool's size (default: what all requests need at once; with fewer
    a prompt waits until its pages are free).
    Raises DDTreeError for a row of logits without a token to draw (all NaN or -inf)."""
    dev = runner.device
    if chunk_tokens < len(prompts):
        raise ValueError("chunk_tokens must leave every request a token")
    if max_new_tokens < 1 or any(p.numel() < 1 for p in prompts):
        raise ValueError("every prompt and answer has at least one token")
    R = len(prompts)
    ids = [p.reshape(-1).tolist() for p in prompts]
    most = [-(-(len(p) + max_new_tokens) // page_size) for p in ids]  # pages at its longest
    if n_pages is None:
        n_pages = sum(most)
    if n_pages < max(most):
        raise ValueError(f"{n_pages} pages cannot hold the longest request ({max(most)})")
    cache = PagedKVCache(len(runner.layers), n_pages, runner.kv_heads, runner.head_dim, R,
                         max(most), page_size, dev)
    stop = set(stop_token_ids or ())
    length = [0] * R                      # rows in the cache
    answer: list[list[int]] = [[] for _ in range(R)]
    admitted, ended = [False] * R, [False] * R

    def rules(n):
        full = lambda v, dt: torch.full((n,), v, dtype=dt, device=dev)  # noqa: E731
        return dict(temperature=full(temperature, torch.float32),
                    top_k=full(top_k, torch.int32), top_p=full(top_p, torch.float32),
                    min_p=full(min_p, torch.float32))

    while not all(ended):
        # admit prompts whose pages fit beside those the running requests may still need
        held = sum(m for m, a, e in zip(most, admitted, ended) if a and not e)
        for r in range(R):
            if not admitted[r] and held + most[r] <= n_pages:
                admitted[r] = True
                held += most[r]
        running = [r for r in range(R) if admitted[r] and not ended[r]]
        # decoding requests first, one token each; then chunks of the prompts
        new = [0] * R
        room = chunk_tokens
        for r in running:
            if length[r] >= len(ids[r]):
                new[r] = 1
                room -= 1
        for r in running:
            if length[r] < len(ids[r]):
                new[r] = min(room, len(ids[r]) - length[r])
                room -= new[r]
        feed, rows, drawn = [], [], []
        for r in range(R):
            if new[r] == 0:
                continue
            seq = ids[r] + answer[r]
            feed += seq[length[r]:length[r] + new[r]]
            if length[r] + new[r] == len(seq):  # the row whose next token is not known yet
                rows.append(len(feed) - 1)
                drawn.append(r)
        target = [0 if ended[r] else length[r] + new[r] for r in range(R)]
        step = cache.step(torch.tensor(target, dtype=torch.int32, device=dev), len(feed))
        logits = runner.forward_paged(torch.tensor(feed, dtype=torch.int64, device=dev), cache, step,
                                      max(new), torch.tensor(rows, dtype=torch.int64, device=dev))
        length = target
        if drawn:
            u = torch.rand(len(drawn), device=dev, generator=generator)
            tokens, _ = K.sample(logits, u, **rules(len(drawn)))
            for r, t in zip(drawn, tokens.tolist()):
                if t < 0:
                    raise _lib.DDTreeError(f"request {r}: no token to draw after {len(answer[r])} "
                                           "(its logits are all NaN or -inf)")
                answer[r].append(t)
                ended[r] = len(answer[r]) >= max_new_tokens or t in stop
        cache.check()
    return [torch.tensor(a, dtype=torch.int64) for a in answer]
