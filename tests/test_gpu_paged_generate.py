"""The paged serving path: Qwen3VerifyRunner.forward_paged over PagedKVCache (prompts in chunks,
decoded tokens, rolled-back rows, several requests in one forward) against the contiguous
forward of the same runner, and paged_generate's answers against it."""
import copy

import numpy as np
import pytest
import torch

from mdflash_b200 import _lib
from mdflash_b200 import kernels as K
from mdflash_b200.cache import TreeKVCache
from mdflash_b200.paged import PagedKVCache, paged_generate

pytestmark = pytest.mark.gpu
V, TOL = 2048, 2e-2


@pytest.fixture(scope="module")
def models(cuda_device):
    from transformers import Qwen3Config, Qwen3ForCausalLM
    from mdflash_b200.runner import Qwen3VerifyRunner
    cfg = Qwen3Config(vocab_size=V, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                      rope_theta=1e6, max_position_embeddings=4096, rms_norm_eps=1e-6,
                      tie_word_embeddings=False, initializer_range=0.2)
    torch.manual_seed(1)
    model = Qwen3ForCausalLM(cfg).to(cuda_device, torch.bfloat16).eval()
    exact = copy.deepcopy(model).float()
    exact.config._attn_implementation = "eager"
    return Qwen3VerifyRunner(model), exact


@pytest.fixture(scope="module")
def runner(models):
    return models[0]


def _contiguous(runner, dev, ids):
    """Logits of every row of one sequence, one causal forward."""
    cache = TreeKVCache(2, len(ids) + 1).allocate(2, 128, torch.bfloat16, dev)
    with torch.inference_mode():
        return runner.forward(torch.tensor(ids, device=dev), torch.arange(len(ids), device=dev),
                              cache, 0, None, causal=True)


def _row_errors(got, truth):
    """Relative 2-norm error of every row of logits."""
    return ((got.float() - truth).norm(dim=-1) / truth.norm(dim=-1)).cpu()


@pytest.mark.parametrize("page", [16, 64])
def test_forward_paged_matches_contiguous_forward(cuda_device, models, page):
    """Three requests, steps of different kinds: whole prompts, chunks, single tokens, an idle
    place, and a rollback after which other tokens are fed.  The truth is the same weights' fp32
    forward.  A bf16 forward of this model is 1 to 2% off it whichever path runs it; the paged
    path rounds no more often than the contiguous one, so over all rows its mean error is at
    most 1.25 times the contiguous path's, and no row is off by more than twice that path's worst
    row (a wrong row is off by about 140%)."""
    dev = cuda_device
    runner, exact = models
    rng = np.random.default_rng(3)
    seq = [[int(t) for t in rng.integers(0, V, 400)] for _ in range(3)]
    other = [int(t) for t in rng.integers(0, V, 400)]
    cache = PagedKVCache(2, 64 if page == 16 else 20, 2, 128, 3, 26 if page == 16 else 7, page, dev)
    lens = [0, 0, 0]

    def both(ids):
        with torch.inference_mode():
            truth = exact(torch.tensor([ids], device=dev)).logits[0]
        return truth, _row_errors(_contiguous(runner, dev, ids), truth)

    refs = [both(s) for s in seq]
    #        target lengths of a step
    steps = [[100, 0, 7], [101, 133, 8], [180, 134, 9], [181, 135, 9], [200, 300, 10], [190, 301, 11],
             [191, 302, 300]]
    mine, theirs = [], []
    for target in steps:
        new = [max(t - o, 0) for t, o in zip(target, lens)]
        if target[0] < lens[0]:  # rolled back: the sequence goes on with other tokens
            seq[0] = seq[0][:target[0]] + other[target[0]:]
            refs[0] = both(seq[0])
        feed = [t for r in range(3) for t in seq[r][lens[r]:lens[r] + new[r]]]
        st = cache.step(torch.tensor(target, dtype=torch.int32, device=dev), sum(new) + 3)
        with torch.inference_mode():
            got = runner.forward_paged(torch.tensor(feed, device=dev), cache, st, max(new))
        at = 0
        for r in range(3):
            rows = slice(lens[r], lens[r] + new[r])
            mine.append(_row_errors(got[at:at + new[r]], refs[r][0][rows]))
            theirs.append(refs[r][1][rows])
            at += new[r]
        lens = target
    cache.check()
    mine, theirs = torch.cat(mine), torch.cat(theirs)
    print(f"[paged] row error mean {mine.mean():.4f} max {mine.max():.4f}, contiguous "
          f"{theirs.mean():.4f} {theirs.max():.4f}")
    assert float(mine.mean()) <= 1.25 * float(theirs.mean())
    assert float(mine.max()) <= 2 * float(theirs.max())
    held = sum(-(-n // page) for n in lens)
    assert int(cache.free_count.item()) == cache.n_pages - held


def test_paged_generate_greedy_follows_the_contiguous_model(cuda_device, runner):
    """Every greedy token is the contiguous forward's argmax, or within the logits' tolerance
    of it; waiting for pages (a small pool) and other chunk sizes give the same answers where
    no near-tie decides."""
    dev = cuda_device
    rng = np.random.default_rng(5)
    prompts = [torch.from_numpy(rng.integers(0, V, n)) for n in (5, 130, 64, 1, 300)]
    out = paged_generate(runner, prompts, 12, chunk_tokens=64, page_size=16)
    assert [o.numel() for o in out] == [12] * 5
    for p, o in zip(prompts, out):
        logits = _contiguous(runner, dev, p.tolist() + o.tolist()).float()[p.numel() - 1:-1]
        best = logits.amax(-1)
        mine = logits.gather(1, o.to(dev)[:, None])[:, 0]
        assert bool((mine >= best - 2 * TOL * best.abs()).all())
    small = paged_generate(runner, prompts, 12, chunk_tokens=512, page_size=32, n_pages=11)
    same = sum(int((a == b).sum()) for a, b in zip(out, small))
    print(f"[paged] {same} of 60 tokens equal with another pool and chunk size")


def test_paged_generate_samples_reproducibly_and_stops(cuda_device, runner):
    dev = cuda_device
    prompts = [torch.arange(9), torch.arange(40)]
    kw = dict(temperature=0.9, top_k=40, top_p=0.95)
    a = paged_generate(runner, prompts, 20, generator=torch.Generator(dev).manual_seed(3), **kw)
    b = paged_generate(runner, prompts, 20, generator=torch.Generator(dev).manual_seed(3), **kw)
    c = paged_generate(runner, prompts, 20, generator=torch.Generator(dev).manual_seed(4), **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert any(not torch.equal(x, y) for x, y in zip(a, c))
    stop = int(a[0][7])
    first = a[0].tolist().index(stop)
    d = paged_generate(runner, prompts[:1], 20, stop_token_ids=[stop], **kw,
                       generator=torch.Generator(dev).manual_seed(3))
    assert d[0].numel() <= 20 and (d[0].numel() == 20 or int(d[0][-1]) == stop)
    assert first <= 7


@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
@pytest.mark.parametrize("step", [0, 2])
def test_paged_generate_reports_a_row_without_a_token(cuda_device, runner, bad, step):
    """Logits of one request that hold nothing to draw, in the first step or in a later one, raise
    an error on the host; the row's -1 is not fed to the embedding."""

    class Broken:
        steps = 0

        def __getattr__(self, name):
            return getattr(runner, name)

        def forward_paged(self, ids, *args):
            assert int(ids.min()) >= 0
            logits = runner.forward_paged(ids, *args)
            if self.steps == step:
                logits[1] = bad
            self.steps += 1
            return logits

    broken = Broken()
    with pytest.raises(_lib.DDTreeError, match="request 1: no token to draw"):
        paged_generate(broken, [torch.arange(9), torch.arange(40)], 6)
    assert broken.steps == step + 1


def test_recorded_decode_step_serves_growing_requests(cuda_device, runner):
    """Page tables, forward and sampling of a decode step recorded in one graph, replayed while
    the requests grow across pages: the tokens of the eager loop."""
    dev = cuda_device
    prompts = [torch.arange(30), torch.arange(7), torch.arange(64)]
    want = paged_generate(runner, prompts, 24, page_size=16)
    cache = PagedKVCache(2, 24, 2, 128, 3, 8, 16, dev)
    ids = torch.cat(prompts).to(dev)
    step = cache.step(torch.tensor([30, 7, 64], dtype=torch.int32, device=dev), 101)
    f32 = dict(dtype=torch.float32, device=dev)
    u, temp = torch.zeros(3, **f32), torch.zeros(3, **f32)
    with torch.inference_mode():
        logits = runner.forward_paged(ids, cache, step, 64, torch.tensor([29, 36, 100], device=dev))
        token = K.sample(logits, u, temp)[0].clone()
        got = [token.tolist()]

        def decode():
            st = cache.step(cache.lens + 1, 3)
            K.sample(runner.forward_paged(token, cache, st, 1), u, temp, out=token)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warms up and decodes one token
            decode()
        torch.cuda.current_stream().wait_stream(side)
        got.append(token.tolist())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            decode()
        for _ in range(22):
            graph.replay()
            got.append(token.tolist())
    cache.check()
    assert cache.lens.tolist() == [53, 30, 87]
    assert [list(t) for t in zip(*got)] == [w.tolist() for w in want]


def test_paged_cache_reports_an_exhausted_pool(cuda_device):
    cache = PagedKVCache(1, 4, 1, 128, 2, 8, 16, cuda_device)
    st = cache.step(torch.tensor([40, 60], dtype=torch.int32, device=cuda_device), 100)
    with pytest.raises(_lib.DDTreeError, match="page-table step refused"):
        cache.check()
    assert st.kv_lens.tolist() == [0, 0] and int(cache.free_count.item()) == 4
    assert int((st.slot_map >= 0).sum()) == 0
    # the refused step's attention has no rows to compute
    q = torch.ones((2, 1, 128), dtype=torch.bfloat16, device=cuda_device)
    out = K.paged_attention(q, cache.k_pages[0], cache.v_pages[0], cache.block_table, st.cu_new,
                            st.kv_lens, 60, out=torch.full_like(q, 5.0), status=cache.status)
    cache.check()
    assert bool((out == 5).all())


def test_paged_generate_refusals(cuda_device, runner):
    p = [torch.arange(4), torch.arange(4)]
    with pytest.raises(ValueError):
        paged_generate(runner, p, 4, chunk_tokens=1)
    with pytest.raises(ValueError):
        paged_generate(runner, p, 0)
    with pytest.raises(ValueError):
        paged_generate(runner, p, 100, n_pages=2)
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 1, 128, 2, 8, 24, cuda_device)
