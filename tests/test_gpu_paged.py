"""The paged K/V cache's kernels against plain 64-bit implementations: ddt_page_tables (exact,
against a request-by-request restatement on the host), ddt_paged_qk_norm_rope and
ddt_paged_attn (element-wise bounds derived from their roundings).  No counterpart in the
reference, which keeps one contiguous cache per request (ddtree.py:387)."""
import math

import numpy as np
import pytest
import torch

from mdflash_b200 import _lib
from mdflash_b200 import kernels as K

pytestmark = pytest.mark.gpu

D = 128
EPS = 1e-6


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _pages(n, page):
    return -(-n // page)


# ---- page tables -------------------------------------------------------------------------
def _tables_ref(old, new, table, free, count, page, max_tokens):
    """The step on host lists; None when it does not fit."""
    table, stack = [list(r) for r in table], list(free[:count])
    mx = len(table[0])
    if any(x < 0 for x in old + new) or any(_pages(x, page) > mx for x in old + new):
        return None
    for r, (o, n) in enumerate(zip(old, new)):
        for j in range(_pages(n, page), _pages(o, page)):
            stack.append(table[r][j])
    if len(stack) > len(free):
        return None
    pushed = list(stack)
    slots, pos, cu = [], [], [0]
    for r, (o, n) in enumerate(zip(old, new)):
        for j in range(_pages(o, page), _pages(n, page)):
            if not stack:
                return None
            table[r][j] = stack.pop()
        for p in range(o, n):
            pos.append(p)
            slots.append(table[r][p // page] * page + p % page)
        cu.append(len(pos))
    if len(pos) > max_tokens:
        return None
    pad = max_tokens - len(pos)
    free = pushed + list(free[len(pushed):])
    return dict(kv_lens=new, cu_new=cu, slot_map=slots + [-1] * pad, positions=pos + [0] * pad,
                free_count=[len(stack)], block_table=table, free_pages=free)


def _tables_case(rng, R, page, max_pages, kinds):
    top = page * max_pages
    old, new = [], []
    for _ in range(R):
        kind = rng.choice(kinds)
        o = int(rng.integers(0, top + 1))
        n = {"grow1": min(o + 1, top), "grow": int(rng.integers(o, top + 1)),
             "shrink": int(rng.integers(0, o + 1)), "end": 0, "same": o,
             "fresh": int(rng.integers(0, top + 1))}[kind]
        if kind == "fresh":
            o = 0
        old.append(o)
        new.append(n)
    return old, new


def _run_tables(dev, old, new, page, max_pages, spare, max_tokens, seed=0, in_place=False):
    rng = np.random.default_rng(seed)
    used = sum(_pages(max(o, 0), page) for o in old)
    ids = rng.permutation(used + spare).tolist()
    table, at = [], 0
    for o in old:
        k = _pages(max(o, 0), page)
        table.append((ids[at:at + k] + [-7] * max_pages)[:max_pages])
        at += k
    free = ids[used:] + [-9] * used
    ref = _tables_ref(old, new, table, free, spare, page, max_tokens)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    t = dict(old=_i32(old, dev), new=_i32(new, dev), table=_i32(table, dev), free=_i32(free, dev),
             count=_i32([spare], dev))
    out = None
    if in_place:
        out = K.PageStep.allocate(dev, len(old), max_tokens)
        out.kv_lens, out.free_count = t["old"], t["count"]
    step = K.page_tables(t["old"], t["new"], t["table"], t["free"], t["count"], page, max_tokens,
                         out=out, status=status)
    got = dict(kv_lens=step.kv_lens, cu_new=step.cu_new, slot_map=step.slot_map,
               positions=step.positions, free_count=step.free_count, block_table=t["table"],
               free_pages=t["free"])
    if ref is None:
        assert int(status.item()) == K.STATUS_PAGES
        ref = dict(kv_lens=old, cu_new=[0] * (len(old) + 1), slot_map=[-1] * max_tokens,
                   positions=[0] * max_tokens, free_count=[spare], block_table=table,
                   free_pages=free)
        fits = False
    else:
        assert int(status.item()) == 0
        fits = True
    for name, want in ref.items():
        assert torch.equal(got[name].cpu().long(), torch.tensor(want, dtype=torch.int64)
                           .reshape(got[name].shape)), name
    return fits


@pytest.mark.parametrize("R,page,max_pages,kinds", [
    (1, 16, 1, ["fresh"]), (1, 16, 8, ["grow1"]), (3, 16, 5, ["same"]),
    (7, 32, 9, ["grow", "shrink", "end", "fresh"]), (64, 16, 33, ["grow1"]),
    (129, 64, 4, ["grow1", "shrink", "end"]), (1000, 16, 7, ["grow", "shrink", "end", "same"]),
    (2048, 16, 3, ["grow", "shrink", "end", "fresh"]), (5, 1024, 2, ["grow", "shrink"]),
    (33, 128, 40, ["fresh", "end"])])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_tables_match_restatement(cuda_device, R, page, max_pages, kinds, in_place):
    rng = np.random.default_rng(R * 7 + page)
    old, new = _tables_case(rng, R, page, max_pages, kinds)
    tokens = sum(max(n - o, 0) for o, n in zip(old, new))
    grown = sum(max(_pages(n, page) - _pages(o, page), 0) for o, n in zip(old, new))
    assert _run_tables(cuda_device, old, new, page, max_pages, grown + 1, tokens + 5, R, in_place)


def test_page_tables_take_pages_given_back_in_the_same_step(cuda_device):
    # an empty stack: the growing request lives on what the others give back
    assert _run_tables(cuda_device, [64, 0, 48], [16, 80, 16], 16, 6, 0, 80)
    assert _run_tables(cuda_device, [64, 0, 48], [0, 112, 0], 16, 7, 0, 112)


def test_page_tables_of_requests_without_pages(cuda_device):
    # nothing held, nothing wanted, and a free stack of no entries at all
    assert _run_tables(cuda_device, [0, 0, 0], [0, 0, 0], 16, 3, 0, 0)
    assert not _run_tables(cuda_device, [0, 0, 0], [0, 1, 0], 16, 3, 0, 4)


@pytest.mark.parametrize("old,new,spare,max_tokens", [
    ([10, 20], [60, 70], 5, 200),    # 6 pages wanted, 5 free
    ([10, 20], [12, 200], 50, 300),  # beyond max_pages
    ([10, -1], [12, 3], 50, 300), ([10, 0], [12, -3], 50, 300),  # negative lengths
    ([10, 0], [12, 30], 50, 31)])    # more new tokens than announced
@pytest.mark.parametrize("in_place", [False, True])
def test_page_tables_refuse_a_step_that_does_not_fit(cuda_device, old, new, spare, max_tokens,
                                                     in_place):
    assert not _run_tables(cuda_device, old, new, 16, 8, spare, max_tokens, in_place=in_place)


def test_page_tables_status_is_reported(cuda_device):
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    K.page_tables(_i32([0], cuda_device), _i32([40], cuda_device),
                  torch.zeros((1, 4), dtype=torch.int32, device=cuda_device),
                  torch.zeros(4, dtype=torch.int32, device=cuda_device), _i32([2], cuda_device),
                  16, 64, status=status)
    with pytest.raises(_lib.DDTreeError, match="page-table step refused"):
        K.check_status(status, "ddt_page_tables")
    assert int(status.item()) == 0


# ---- K / V write ---------------------------------------------------------------------------
def _pool(n_pages, heads, page, layout, dev, fill=float("nan")):
    shape = (n_pages, heads, page, D) if layout == "heads_first" else (n_pages, page, heads, D)
    t = torch.full(shape, fill, dtype=torch.bfloat16, device=dev)
    return t if layout == "heads_first" else t.permute(0, 2, 1, 3)


def _rope(positions, theta=1e6):
    inv = theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = positions.double()[:, None] * inv
    cos, sin = ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)
    words = (cos.view(torch.int16).to(torch.int32) & 0xffff) | (sin.view(torch.int16).to(torch.int32) << 16)
    return words, cos.double(), sin.double()


@pytest.mark.parametrize("T,hq,hkv,page,layout,extra", [
    (1, 32, 8, 16, "heads_first", 0), (2, 1, 1, 32, "tokens_first", 0),
    (17, 16, 8, 16, "tokens_first", 0), (63, 8, 2, 64, "heads_first", 8),
    (129, 40, 8, 128, "heads_first", 0), (1000, 5, 1, 1024, "tokens_first", 128),
    (301, 3, 3, 256, "heads_first", 16)])
def test_paged_write_matches_formula(cuda_device, T, hq, hkv, page, layout, extra):
    """Every element within its own bf16 rounding (half a step, 2^-8 relative to be safe at the
    step's lower end) plus fp32 arithmetic on the two products (a few 2^-24 of their sizes);
    V exact; rows of the pool that no slot names, and slots of -1, untouched."""
    g = torch.Generator().manual_seed(T)
    x = (torch.randn((T, (hq + 2 * hkv) * D + extra), generator=g) * 3).to(torch.bfloat16)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2))
    n_pages = _pages(T, page) + 2
    slots = torch.randperm(n_pages * page, generator=g)[:T]
    slots[T // 2] = -1
    pos = torch.randint(0, 40000, (T,), generator=g)
    words, cos, sin = _rope(pos)
    kp, vp = (_pool(n_pages, hkv, page, layout, cuda_device) for _ in range(2))
    qkv = x.to(cuda_device)[:, :(hq + 2 * hkv) * D]
    q = K.paged_qk_norm_rope(qkv, qw.to(cuda_device), kw.to(cuda_device), words.to(cuda_device),
                             slots.to(cuda_device), kp, vp, EPS)
    h = x[:, :(hq + 2 * hkv) * D].double().view(T, -1, D)
    w = torch.cat([qw.double().expand(hq, D), kw.double().expand(hkv, D)])
    y = h[:, :hq + hkv]
    y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
    a, b = y[..., :64], y[..., 64:]
    c, s = cos[:, None], sin[:, None]
    ref = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    tol = ref.abs() * 2.0 ** -8 + size * 2.0 ** -20
    assert bool(((q.cpu().double() - ref[:, :hq]).abs() <= tol[:, :hq]).all())
    wrote = torch.zeros(n_pages * page, dtype=torch.bool)
    kc, vc = kp.cpu().double(), vp.cpu().double()
    for t in range(T):
        sl = int(slots[t])
        if sl < 0:
            continue
        wrote[sl] = True
        assert bool(((kc[sl // page, :, sl % page] - ref[t, hq:]).abs() <= tol[t, hq:]).all())
        assert torch.equal(vc[sl // page, :, sl % page], h[t, hq + hkv:])
    rest = (~wrote).view(n_pages, page)
    for t in (kc, vc):
        assert bool(t.permute(0, 2, 1, 3)[rest].isnan().all())


def test_paged_write_zero_rows_and_slots_outside(cuda_device):
    """A zero head gives zeros (the epsilon carries the root); slots outside the pool write
    nothing; no tokens is no work."""
    kp, vp = (_pool(2, 1, 16, "heads_first", cuda_device) for _ in range(2))
    w = torch.ones(D, dtype=torch.bfloat16, device=cuda_device)
    words = _rope(torch.arange(3))[0].to(cuda_device)
    qkv = torch.zeros((3, 3 * D), dtype=torch.bfloat16, device=cuda_device)
    slots = torch.tensor([32, 1 << 40, -(1 << 40)], device=cuda_device)
    q = K.paged_qk_norm_rope(qkv, w, w, words, slots, kp, vp)
    assert bool((q == 0).all()) and bool(kp.isnan().all()) and bool(vp.isnan().all())
    assert K.paged_qk_norm_rope(qkv[:0], w, w, words[:0], slots[:0], kp, vp).shape == (0, 1, D)


def test_paged_write_refuses_rows_that_overlap(cuda_device):
    """One projection row expanded to several tokens, or rows closer than their width, are
    refused; the stride of a single row does not matter."""
    kp, vp = (_pool(2, 1, 16, "heads_first", cuda_device) for _ in range(2))
    w = torch.ones(D, dtype=torch.bfloat16, device=cuda_device)
    words = _rope(torch.arange(3))[0].to(cuda_device)
    slots = torch.arange(3, device=cuda_device)
    one = torch.randn((1, 3 * D), device=cuda_device).to(torch.bfloat16)
    for qkv in (one.expand(3, -1), torch.zeros(9 * D, dtype=torch.bfloat16, device=cuda_device)
                .as_strided((3, 3 * D), (2 * D, 1))):
        with pytest.raises(_lib.DDTreeError):
            K.paged_qk_norm_rope(qkv, w, w, words, slots, kp, vp)
    q = K.paged_qk_norm_rope(one, w, w, words[:1], slots[:1], kp, vp)
    k, v = kp[0, :, 0].clone(), vp[0, :, 0].clone()
    q2 = K.paged_qk_norm_rope(one.as_strided((1, 3 * D), (7, 1)), w, w, words[:1], slots[1:2], kp, vp)
    assert torch.equal(q, q2) and torch.equal(kp[0, :, 1], k) and torch.equal(vp[0, :, 1], v)


# ---- attention -------------------------------------------------------------------------------
class _Case:
    """Requests with random K / V in a shuffled pool; whatever lies outside their rows is NaN,
    and table entries past their pages name no page."""

    def __init__(self, dev, lens, news, hq, hkv, page, layout="heads_first", seed=0, qscale=1.0,
                 vmean=0.0, fused_q=False, spare_cols=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.news, self.hq, self.hkv, self.page = lens, news, hq, hkv, page
        n_pages = sum(_pages(n, page) for n in lens) + 2
        cols = max([_pages(n, page) for n in lens] + [1]) + spare_cols
        order = torch.randperm(n_pages, generator=g).tolist()
        self.k_pages, self.v_pages = (_pool(n_pages, hkv, page, layout, dev) for _ in range(2))
        table = torch.full((len(lens), cols), 1 << 30, dtype=torch.int32)
        self.keys, self.values = [], []
        at = 0
        for r, n in enumerate(lens):
            k = torch.randn((n, hkv, D), generator=g).to(torch.bfloat16)
            v = (torch.randn((n, hkv, D), generator=g) + vmean).to(torch.bfloat16)
            self.keys.append(k.double().to(dev))
            self.values.append(v.double().to(dev))
            for j in range(_pages(n, page)):
                pg = order[at]
                at += 1
                table[r, j] = pg
                rows = min(page, n - j * page)
                for pool, src in ((self.k_pages, k), (self.v_pages, v)):
                    pool[pg, :, :rows] = src[j * page:j * page + rows].transpose(0, 1).to(dev)
        self.table = table.to(dev)
        cu = np.concatenate([[0], np.cumsum(news)]).astype(int).tolist()
        self.cu = cu
        T = cu[-1]
        q = (torch.randn((T, hq, D), generator=g) * qscale).to(torch.bfloat16)
        self.q64 = q.double().to(dev)
        if fused_q:  # the query heads of a fused projection
            wide = torch.full((T, hq + 2 * hkv, D), float("nan"), dtype=torch.bfloat16, device=dev)
            wide[:, :hq] = q.to(dev)
            self.q = wide[:, :hq]
        else:
            self.q = q.to(dev)
        self.cu_new, self.kv_lens = _i32(cu, dev), _i32(lens, dev)

    def run(self, **kw):
        return K.paged_attention(self.q, self.k_pages, self.v_pages, self.table, self.cu_new,
                                 self.kv_lens, kw.pop("max_new", max(self.news + [0])), **kw)

    def check(self, out, scale=None):
        """|out - ref| <= half a bf16 step of ref, and per key half a bf16 step of its softmax
        weight (a matrix product takes the weights in bf16) times |v|, plus 2^-11 of sum p |v| for
        the scores' fp32 sums and an exponential good to 1.1e-4.  bf16 has 8 significant bits:
        between 2^e and 2^(e+1) its step is 2^(e-7), so half a step is up to 2^-8 of the value."""
        scale = D ** -0.5 if scale is None else scale
        g = self.hq // self.hkv
        for r, (n, new) in enumerate(zip(self.lens, self.news)):
            if new == 0:
                continue
            q = self.q64[self.cu[r]:self.cu[r + 1]].view(new, self.hkv, g, D)
            s = torch.einsum("ihgd,jhd->hgij", q, self.keys[r]) * scale
            i, j = torch.arange(new, device=s.device)[:, None], torch.arange(n, device=s.device)
            s = s.masked_fill(j > n - new + i, -math.inf)
            top = s.amax(-1, keepdim=True) if n else s.new_full(s.shape[:-1] + (1,), -math.inf)
            p = (s - torch.where(top > -math.inf, top, 0.0)).exp()
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            ref = torch.einsum("hgij,jhd->ihgd", p, self.values[r]).reshape(new, self.hq, D)
            mag = torch.einsum("hgij,jhd->ihgd", p, self.values[r].abs()).reshape(new, self.hq, D)
            tol = ref.abs() * 2.0 ** -8 + mag * (2.0 ** -8 + 2.0 ** -11) + 1e-30
            got = out[self.cu[r]:self.cu[r + 1]].double()
            bad = ~((got - ref).abs() <= tol)
            assert not bool(bad.any()), (r, n, new, int(bad.sum()),
                                         float(((got - ref).abs() / tol)[bad].nan_to_num(9e9).max()))


ATTN = {
    # lens, new, q heads, kv heads, page
    "one_key": ([1], [1], 32, 8, 16),
    "no_key": ([0, 5], [1, 1], 32, 8, 16),
    "rows_before_the_first_key": ([3, 40], [7, 40], 8, 2, 16),
    "idle_requests": ([17, 0, 33, 64], [0, 0, 1, 0], 16, 8, 32),
    "page_ends": ([15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257], [1] * 12, 32, 8, 16),
    "page_ends_chunks": ([63, 64, 65, 127, 128, 129, 300], [63, 64, 3, 127, 128, 5, 299], 8, 4, 64),
    "decode_mix": ([1, 7000, 300, 1025, 63, 4096], [1] * 6, 32, 8, 16),
    "decode_page_1024": ([1, 7000, 300, 1025, 1024], [1] * 5, 16, 8, 1024),
    "long_decode": ([40001], [1], 32, 8, 16),
    "group_1": ([200, 77], [1, 9], 4, 4, 16),
    "group_3": ([500, 129, 64], [1, 20, 64], 6, 2, 16),
    "group_5": ([500, 131], [43, 1], 10, 2, 32),
    "group_7_chunk": ([900], [333], 14, 2, 64),
    "group_16": ([700, 65], [3, 5], 32, 2, 128),
    "group_64": ([257, 20], [2, 20], 64, 1, 16),
    "one_kv_head": ([3000, 2], [5, 2], 8, 1, 256),
    "blocks_of_16": ([700, 16, 2500, 1000], [16, 16, 16, 16], 32, 8, 32),
    "blocks_of_17": ([700, 17, 2501], [17, 17, 16], 32, 8, 32),
    "prompt": ([1000], [1000], 32, 8, 16),
    "prompt_chunk": ([3001], [513], 16, 8, 16),
    "prompt_chunks": ([2048, 700, 1300, 257], [600, 700, 65, 256], 32, 8, 64),
    "chunk_among_decodes": ([900, 5000, 64, 1, 777], [1, 400, 1, 1, 1], 16, 8, 16),
    "chunk_page_512": ([1500, 513], [512, 100], 8, 8, 512),
    "many_requests": (list(range(1, 301)), [1] * 300, 8, 2, 16),
    # both kernels: a chunk, single tokens, idle places and a request of 20 rows between them
    "chunk_among_30": ([37 * i + 1 for i in range(15)] + [700, 0, 64] + [50 * i + 9 for i in range(13)],
                       [1] * 15 + [300, 0, 10] + [1] * 13, 16, 8, 16),
}


@pytest.mark.parametrize("name", ATTN)
def test_paged_attention_matches_formula(cuda_device, name):
    lens, news, hq, hkv, page = ATTN[name]
    c = _Case(cuda_device, lens, news, hq, hkv, page, seed=len(name))
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    c.check(c.run(status=status))
    assert int(status.item()) == 0


@pytest.mark.parametrize("name", ["decode_mix", "blocks_of_16", "prompt_chunks", "page_ends_chunks"])
def test_paged_attention_layouts_and_strides(cuda_device, name):
    """Token-major pages, the query heads of a fused projection, a wider table, an output with
    strides of its own; the surroundings of the output stay as they were."""
    lens, news, hq, hkv, page = ATTN[name]
    c = _Case(cuda_device, lens, news, hq, hkv, page, layout="tokens_first", seed=5, fused_q=True,
              spare_cols=3)
    T = c.cu[-1]
    wide = torch.full((T + 1, hq + 1, D + 8), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out = wide[:T, 1:, :D]
    c.run(out=out)
    c.check(out)
    assert bool((wide[T] == 7).all()) and bool((wide[:, 0] == 7).all()) and \
        bool((wide[..., D:] == 7).all())


@pytest.mark.parametrize("name", ["decode_mix", "blocks_of_17", "prompt_chunks"])
@pytest.mark.parametrize("qscale,scale", [(30.0, None), (1.0, 1.0), (0.0, None), (1.0, 0.0)])
def test_paged_attention_sharp_and_flat_scores(cuda_device, name, qscale, scale):
    """Scores of a hundred (one key takes it all) down to all equal, and V with a mean, so that
    the bound is relative to a result that does not cancel."""
    lens, news, hq, hkv, page = ATTN[name]
    c = _Case(cuda_device, lens, news, hq, hkv, page, seed=9, qscale=qscale, vmean=1.0)
    out = c.run(scale=scale)
    c.check(out, scale=scale)


@pytest.mark.parametrize("hq,hkv,new", [(8, 8, 1), (8, 8, 8), (6, 2, 2), (16, 8, 4), (32, 8, 2),
                                        (10, 2, 1), (16, 2, 1)])
def test_paged_attention_weights_of_few_rows(cuda_device, hq, hkv, new):
    """Up to 8 query rows per (request, KV head) take the softmax weights as two bf16 parts: the
    first is off by at most 2^-8 of the weight (half a bf16 step), the second by 2^-8 of that.  So an
    element is off by half a bf16 step of itself, 2^-16 of sum p |v|, and 2^-11 of it for the scores'
    fp32 sums: 128 products of at most 12 in all, 2^-23 each, in numerator and sum.  Few keys,
    where the roundings of the weights do not average out, up to many."""
    rng = np.random.default_rng(hq)
    lens = [int(n) for n in rng.integers(new, 12, 60)] + [70, 300, 5000]
    c = _Case(cuda_device, lens, [new] * len(lens), hq, hkv, 16, seed=hq + new)
    out = c.run()
    g = hq // hkv
    for r, n in enumerate(lens):
        q = c.q64[c.cu[r]:c.cu[r + 1]].view(new, hkv, g, D)
        s = torch.einsum("ihgd,jhd->hgij", q, c.keys[r]) * D ** -0.5
        i, j = torch.arange(new, device=s.device)[:, None], torch.arange(n, device=s.device)
        p = s.masked_fill(j > n - new + i, -math.inf).softmax(-1)
        ref, mag = (torch.einsum("hgij,jhd->ihgd", p, v).reshape(new, hq, D)
                    for v in (c.values[r], c.values[r].abs()))
        tol = ref.abs() * 2.0 ** -8 + mag * (2.0 ** -16 + 2.0 ** -11)
        err = (out[c.cu[r]:c.cu[r + 1]].double() - ref).abs()
        assert bool((err <= tol).all()), (r, n, int((err > tol).sum()), float((err / tol).max()))


def test_paged_attention_is_repeatable(cuda_device):
    lens, news, hq, hkv, page = ATTN["chunk_among_decodes"]
    c = _Case(cuda_device, lens, news, hq, hkv, page, seed=3)
    a = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), a)


def test_paged_attention_skips_requests_out_of_range(cuda_device):
    """A request whose lengths cannot be is skipped and reported; the others are computed."""
    lens, news, hq, hkv, page = ATTN["blocks_of_16"]
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for what in ("max_new", "long", "negative"):
        c = _Case(cuda_device, lens, news, hq, hkv, page, seed=4)
        full = c.run()
        out = torch.full_like(full, 3.0)
        kw = {}
        if what == "long":
            c.kv_lens[1] = 1 << 28
        elif what == "negative":
            c.kv_lens[1] = -4
        else:
            c.cu_new[2:] += 1  # request 1 then has one more new token than announced
            c.q = torch.cat([c.q[:32], c.q[:1], c.q[32:]])
            out = torch.full_like(c.q, 3.0)
        c.run(out=out, status=status, max_new=16, **kw)
        assert int(status.item()) == K.STATUS_PAGED_RANGE
        with pytest.raises(_lib.DDTreeError, match="paged request out of range"):
            K.check_status(status, "ddt_paged_attn")
        skip = 17 if what == "max_new" else 16
        c.check(torch.cat([out[:16], full[16:32], out[16 + skip:]]))
        assert bool((out[16:16 + skip] == 3).all())


@pytest.mark.parametrize("hq,hkv", [(17, 1), (32, 1), (64, 1), (128, 2)])
@pytest.mark.parametrize("what", ["prompt_among_idle_places", "decodes_with_a_loose_bound"])
def test_paged_attention_wide_groups_among_many_places(cuda_device, hq, hkv, what):
    """More than 16 query heads per KV head in a batch of many places: the first prompt of an
    otherwise idle server, and decoded tokens whose announced bound is the whole batch."""
    places = 160
    if what == "prompt_among_idle_places":
        lens, news = [0] * places, [0] * places
        lens[70], news[70] = 130, 100
    else:
        lens, news = [3 * i + 1 for i in range(places)], [1] * places
    c = _Case(cuda_device, lens, news, hq, hkv, 16, seed=hq)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    c.check(c.run(max_new=c.cu[-1], status=status))
    assert int(status.item()) == 0


def test_paged_attention_rows_without_request_are_left(cuda_device):
    c = _Case(cuda_device, [70, 9], [3, 2], 8, 2, 16)
    q = torch.cat([c.q, c.q[:4]])
    out = torch.full_like(q, 3.0)
    K.paged_attention(q, c.k_pages, c.v_pages, c.table, c.cu_new, c.kv_lens, 3, out=out)
    c.check(out[:5])
    assert bool((out[5:] == 3).all())


@pytest.mark.parametrize("name", ["decode_mix", "blocks_of_16", "prompt_chunks"])
@pytest.mark.parametrize("wrong", [-1, "past_the_pool", 1 << 30])
def test_paged_attention_reports_pages_outside_the_pool(cuda_device, name, wrong):
    """A table entry inside a request's length that names no page of the pool is reported; the
    other requests are computed."""
    lens, news, hq, hkv, page = ATTN[name]
    c = _Case(cuda_device, lens, news, hq, hkv, page, seed=7)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    right = c.run(status=status)
    assert int(status.item()) == 0
    c.table[1, lens[1] // page // 2] = c.k_pages.shape[0] if wrong == "past_the_pool" else wrong
    out = c.run(status=status)
    assert int(status.item()) == K.STATUS_PAGED_RANGE
    with pytest.raises(_lib.DDTreeError, match="paged request out of range"):
        K.check_status(status, "ddt_paged_attn")
    a, b = c.cu[1], c.cu[2]
    c.check(torch.cat([out[:a], right[a:b], out[b:]]))


def test_paged_attention_far_pages(cuda_device):
    """Page offsets beyond 2^32 elements: the rows of a small cache moved to the end of a pool of
    140,000 pages with 32,768 elements each."""
    lens, news, hq, hkv, page = [100, 333], [1, 20], 32, 8, 16
    c = _Case(cuda_device, lens, news, hq, hkv, page, seed=6)
    n = c.k_pages.shape[0]
    total = 140_000
    near = c.run()
    for attr in ("k_pages", "v_pages"):
        big = torch.empty((total, 2 * hkv, page, D), dtype=torch.bfloat16, device=cuda_device)
        view = big[:, hkv:]
        view[total - n:] = getattr(c, attr)
        setattr(c, attr, view)
    assert (total - n) * c.k_pages.stride(0) > 1 << 32
    table = c.table.clone()
    c.table = torch.where(table < n, table + total - n, table)
    out = c.run()
    assert torch.equal(out, near)
    c.check(out)


def test_paged_kernels_on_two_streams_at_once(cuda_device):
    """Calls that overlap on two streams share no scratch: 30 rounds of cut units and page steps on
    each, all equal to what either gives alone."""
    cases = [_Case(cuda_device, [5000, 3000], [1, 1], 32, 8, 16, seed=1),
             _Case(cuda_device, [4000, 900], [1, 300], 32, 8, 16, seed=2)]
    alone = [c.run() for c in cases]
    lens = [_i32(c.lens, cuda_device) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    steps = [[], []]
    for _ in range(30):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                outs[i].append(c.run())
                steps[i].append(K.page_tables(torch.zeros_like(lens[i]), lens[i], c.table.clone(),
                                              torch.arange(1000, dtype=torch.int32, device=cuda_device),
                                              _i32([1000], cuda_device), 16, 9000))
    torch.cuda.synchronize()
    for i, c in enumerate(cases):
        assert all(torch.equal(o, alone[i]) for o in outs[i])
        for st in steps[i]:
            assert st.kv_lens.tolist() == c.lens and int(st.slot_map.max()) < 16000
            assert int((st.slot_map >= 0).sum()) == sum(c.lens)


@pytest.mark.parametrize("first_cta", [0, 5, 60, 120])
@pytest.mark.parametrize("name", ["long_decode", "cut_blocks", "prompt_chunks", "chunk_among_30"])
def test_paged_attention_wait_timeout_leaves_no_trace(cuda_device, name, first_cta):
    """Every wait of the attention kernels is bounded.  The CTAs from first_cta on withhold their
    loads, so that the waits in them run out (after 2 ms here): the launch returns and sets the
    status word, and the calls after it on the same workspace are right, although units cut between
    these CTAs and the others were left half done."""
    lens, news, hq, hkv, page = ([9000, 7000], [5, 5], 16, 4, 16) if name == "cut_blocks" else ATTN[name]
    c, d = (_Case(cuda_device, lens, news, hq, hkv, page, seed=s, vmean=m)
            for s, m in ((len(name), 0.0), (1, 3.0)))
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    K.paged_attention_wait_check(d.q, d.k_pages, d.v_pages, d.table, d.cu_new, d.kv_lens, max(news),
                                 first_cta, 2_000_000, status)
    torch.cuda.synchronize()
    with pytest.raises(_lib.DDTreeError, match="bounded device wait expired"):
        K.check_status(status, "ddt_paged_attn")
    outs = [c.run(status=status) for _ in range(4)]
    torch.cuda.synchronize()
    K.check_status(status, "ddt_paged_attn")
    c.check(outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_paged_attention_mixed_batch_recorded(cuda_device):
    """Both kernels and the merge in a recorded graph, on a side stream, replayed back to back."""
    lens, news, hq, hkv, page = ATTN["chunk_among_30"]
    c = _Case(cuda_device, lens, news, hq, hkv, page, seed=2)
    eager = c.run()
    c.check(eager)
    outs = [torch.zeros_like(c.q) for _ in range(4)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for o in outs:
            c.run(out=o)
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, eager) for o in outs)


def test_paged_attention_recorded_without_a_first_call_is_refused(cuda_device):
    c = _Case(cuda_device, [70, 9], [3, 2], 8, 2, 16)
    graph = torch.cuda.CUDAGraph()
    with K.WORKSPACES.lane(971):
        with pytest.raises(_lib.DDTreeError, match="before recording"):
            with torch.cuda.graph(graph):
                c.q.add_(0)
                c.run()
        c.run()  # and with one it records
        out = torch.zeros_like(c.q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.run(out=out)
    graph.replay()
    torch.cuda.synchronize()
    c.check(out)


@pytest.mark.parametrize("lane", [0, 5])
def test_paged_kernels_recorded_on_parallel_branches(cuda_device, lane):
    """One recording that forks into three streams and joins them again, each with attention calls
    of cut units and page steps: branches that replay at once share no scratch.  Several replays
    give what the calls give alone, and so does a second recording of the same branches."""
    cases = [_Case(cuda_device, [5000, 3000], [1, 1], 32, 8, 16, seed=1),
             _Case(cuda_device, [4000, 900], [1, 300], 32, 8, 16, seed=2),
             _Case(cuda_device, [7000], [1], 32, 8, 16, seed=3)]
    side = [torch.cuda.Stream() for _ in cases[1:]]
    lens = [_i32(c.lens, cuda_device) for c in cases]
    zero = [torch.zeros_like(n) for n in lens]
    free, count = torch.arange(1000, dtype=torch.int32, device=cuda_device), _i32([1000], cuda_device)
    outs = [[torch.zeros_like(c.q) for _ in range(6)] for c in cases]
    steps = [[K.PageStep.allocate(cuda_device, len(c.lens), 9000) for _ in range(6)] for c in cases]
    tables = [c.table.clone() for c in cases]

    def branch(i):
        for o, step in zip(outs[i], steps[i]):
            cases[i].run(out=o)
            K.page_tables(zero[i], lens[i], tables[i], free, count, 16, 9000, out=step)

    with K.WORKSPACES.lane(lane):
        alone = [c.run() for c in cases]
        for i in range(3):
            branch(i)
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                main = torch.cuda.current_stream()
                for i, st in enumerate(side, 1):
                    st.wait_stream(main)
                    with torch.cuda.stream(st):
                        branch(i)
                branch(0)
                for st in side:
                    main.wait_stream(st)
                cases[1].run(out=outs[1][0])
            for _ in range(5):
                for i in range(3):
                    for o, step in zip(outs[i], steps[i]):
                        o.fill_(7)
                        step.slot_map.fill_(-5)
                graph.replay()
                torch.cuda.synchronize()
                for i, c in enumerate(cases):
                    assert all(torch.equal(o, alone[i]) for o in outs[i])
                    for step in steps[i]:
                        assert step.kv_lens.tolist() == c.lens
                        assert int((step.slot_map >= 0).sum()) == sum(c.lens)
    for i, c in enumerate(cases):
        c.check(outs[i][0])


@pytest.mark.parametrize("news", [[1, 1, 1, 1], [16, 3, 16, 1], [100, 1, 300, 64]])
def test_paged_attention_recorded_once_serves_other_lengths(cuda_device, news):
    """One recorded launch, replayed after the lengths, tables and queries changed; launched on
    a stream that is not the current default."""
    a = _Case(cuda_device, [400, 30, 900, 64], news if max(news) < 65 else [100, 1, 300, 64], 16, 8,
              16, seed=1, spare_cols=80)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(a.q)
    with torch.cuda.stream(stream):
        a.run(out=out)
    torch.cuda.synchronize()
    a.check(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run(out=out)
    for lens in ([401, 31, 901, 65], [500, 1300, 301, 64], [100, 100, 300, 100]):
        b = _Case(cuda_device, lens, news, 16, 8, 16, seed=sum(lens))
        pool = a.k_pages.shape[0]
        keep = b.k_pages.shape[0]
        if keep > pool:
            continue
        for dst, src in ((a.k_pages, b.k_pages), (a.v_pages, b.v_pages)):
            dst.fill_(float("nan"))
            dst[:keep] = src
        a.table.fill_(1 << 30)
        a.table[:, :b.table.shape[1]] = b.table
        a.q.copy_(b.q)
        a.kv_lens.copy_(b.kv_lens)
        graph.replay()
        torch.cuda.synchronize()
        b.check(out)


def test_paged_refusals(cuda_device):
    c = _Case(cuda_device, [70, 9], [3, 2], 8, 2, 16)
    with pytest.raises(ValueError):  # CPU tensors
        K.paged_attention(c.q.cpu(), c.k_pages, c.v_pages, c.table, c.cu_new, c.kv_lens, 3)
    with pytest.raises(ValueError):
        K.paged_attention(c.q.float(), c.k_pages, c.v_pages, c.table, c.cu_new, c.kv_lens, 3)
    with pytest.raises(TypeError):
        K.paged_attention(c.q, c.k_pages.float(), c.v_pages.float(), c.table, c.cu_new, c.kv_lens, 3)
    with pytest.raises(ValueError):
        K.paged_attention(c.q, c.k_pages, c.v_pages[:1], c.table, c.cu_new, c.kv_lens, 3)
    with pytest.raises(ValueError):
        K.paged_attention(c.q, c.k_pages, c.v_pages, c.table.long(), c.cu_new, c.kv_lens, 3)
    with pytest.raises(ValueError):
        K.paged_attention(c.q, c.k_pages, c.v_pages, c.table, c.cu_new[:2], c.kv_lens, 3)
    with pytest.raises(_lib.DDTreeError):  # 7 query heads over 2
        K.paged_attention(c.q[:, :7], c.k_pages, c.v_pages, c.table, c.cu_new, c.kv_lens, 3)
    with pytest.raises(_lib.DDTreeError):  # pages of 24 rows
        odd = torch.zeros((2, 2, 24, D), dtype=torch.bfloat16, device=cuda_device)
        K.paged_attention(c.q, odd, odd, c.table, c.cu_new, c.kv_lens, 3)
    assert K.paged_attention(c.q[:0], c.k_pages, c.v_pages, c.table, c.cu_new, c.kv_lens,
                             0).shape == (0, 8, D)


def test_paged_calls_refuse_what_the_kernels_would_misread(cuda_device):
    c = _Case(cuda_device, [70, 9], [3, 2], 8, 2, 16)
    for status in (torch.zeros(1, dtype=torch.int32),
                   torch.zeros(1, dtype=torch.int64, device=cuda_device),
                   torch.zeros(0, dtype=torch.int32, device=cuda_device)):
        with pytest.raises(ValueError):
            c.run(status=status)
        with pytest.raises(ValueError):
            K.page_tables(_i32([0], cuda_device), _i32([4], cuda_device), _i32([[0]], cuda_device),
                          _i32([0], cuda_device), _i32([1], cuda_device), 16, 4, status=status)
    with pytest.raises(ValueError):
        K.page_tables(_i32([0], cuda_device), _i32([4], cuda_device), _i32([[0]], cuda_device),
                      _i32([0], cuda_device), _i32([1], cuda_device), 16, -1)
    step = K.PageStep.allocate(cuda_device, 1, 3)
    with pytest.raises(ValueError, match="out.slot_map"):  # made for 3 tokens
        K.page_tables(_i32([0], cuda_device), _i32([4], cuda_device), _i32([[0]], cuda_device),
                      _i32([0], cuda_device), _i32([1], cuda_device), 16, 4, out=step)
    w = torch.ones(2 * D, dtype=torch.bfloat16, device=cuda_device)
    rope = torch.zeros((4, D // 2), dtype=torch.int32, device=cuda_device)
    qkv = torch.zeros((4, 12 * D), dtype=torch.bfloat16, device=cuda_device)
    slots = torch.full((4,), -1, dtype=torch.int64, device=cuda_device)
    K.paged_qk_norm_rope(qkv, w[:D], w[:D], rope, slots, c.k_pages, c.v_pages)
    with pytest.raises(ValueError, match="norm weights"):  # every other element
        K.paged_qk_norm_rope(qkv, w[::2], w[:D], rope, slots, c.k_pages, c.v_pages)
    with pytest.raises(ValueError, match="slot"):
        K.paged_qk_norm_rope(qkv, w[:D], w[:D], rope, slots[:3], c.k_pages, c.v_pages)
    with pytest.raises(ValueError, match="out"):
        K.paged_qk_norm_rope(qkv, w[:D], w[:D], rope, slots, c.k_pages, c.v_pages, out=qkv)


def test_paged_calls_recorded_after_other_work(cuda_device):
    """Every call recorded straight after a fill, a copy, a join of two streams and another of the
    calls: launches that may begin before the work in front of them ends still read its results."""
    c = _Case(cuda_device, [900, 70, 41], [1, 1, 1], 16, 4, 16, seed=3)
    d = _Case(cuda_device, [900, 400, 41], [90, 200, 1], 16, 4, 16, seed=4)
    logits = torch.randn((4, 5000), device=cuda_device)
    u = torch.rand(4, device=cuda_device)
    one = torch.ones(4, device=cuda_device)
    token, logprob = K.sample(logits, u, one)
    inputs = [(c.q, c.q.clone()), (d.q, d.q.clone()), (c.kv_lens, c.kv_lens.clone()),
              (d.k_pages, d.k_pages.clone()), (logits, logits.clone())]
    outs = [torch.zeros_like(c.q) for _ in range(2)] + [torch.zeros_like(d.q) for _ in range(2)]
    side = torch.cuda.Stream()

    def blank():
        for t, _ in inputs:
            t.zero_()

    def restore():
        for t, kept in inputs:
            t.copy_(kept)

    def joined():
        blank()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            restore()
        torch.cuda.current_stream().wait_stream(side)

    c.run(out=outs[0])
    d.run(out=outs[0].new_zeros(d.q.shape))
    graph = torch.cuda.CUDAGraph()
    drawn = []
    with torch.cuda.graph(graph):
        blank()
        restore()
        c.run(out=outs[0])
        blank()
        restore()
        d.run(out=outs[2])
        joined()
        c.run(out=outs[1])
        joined()
        d.run(out=outs[3])
        drawn.append(K.sample(logits, u, one))
        joined()
        drawn.append(K.sample(logits, u, one))
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
    torch.cuda.synchronize()
    for o in outs[:2]:
        c.check(o)
    for o in outs[2:]:
        d.check(o)
    for t, lp in drawn:
        assert torch.equal(t, token) and torch.equal(lp, logprob)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_paged_calls_run_on_the_tensors_device():
    """Tensors of a device that is not the current one: every call launches there, on that device's
    current stream, eager and recorded."""
    dev = torch.device("cuda:1")
    with torch.cuda.device(0):
        assert _run_tables(dev, [10, 20], [60, 12], 16, 8, 9, 64)
        c = _Case(dev, [900, 70], [1, 40], 16, 4, 16)
        c.check(c.run())
        out = torch.zeros_like(c.q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.device(dev), torch.cuda.graph(graph):
            with torch.cuda.device(0):
                c.run(out=out)
        graph.replay()
        torch.cuda.synchronize(dev)
        c.check(out)
        x = torch.randn((3, 50), device=dev)
        tok, _ = K.sample(x, torch.rand(3, device=dev), torch.zeros(3, device=dev))
        assert torch.equal(tok, x.argmax(-1))
        w = torch.ones(D, dtype=torch.bfloat16, device=dev)
        kp, vp = (_pool(2, 1, 16, "heads_first", dev) for _ in range(2))
        qkv = torch.randn((2, 3 * D), device=dev).to(torch.bfloat16)
        K.paged_qk_norm_rope(qkv, w, w, _rope(torch.arange(2))[0].to(dev),
                             torch.arange(2, device=dev), kp, vp)
        assert torch.equal(vp[0, 0, :2], qkv[:, 2 * D:])
        assert torch.cuda.current_device() == 0


def test_page_step_outputs_are_ordinary_tensors(cuda_device):
    """They share one allocation: each keeps it alive, and views, copies and torch operations see
    only its own elements."""
    step = K.page_tables(_i32([0, 15], cuda_device), _i32([3, 17], cuda_device),
                         _i32([[-1, -1], [6, -1]], cuda_device), _i32([9, 8, 7], cuda_device),
                         _i32([3], cuda_device), 16, 7)
    kv, cu, slots, pos, count = (step.kv_lens, step.cu_new, step.slot_map, step.positions,
                                 step.free_count)
    del step
    assert [t.dtype for t in (kv, cu, slots, pos, count)] == [torch.int32] * 2 + [torch.int64] * 2 + \
        [torch.int32]
    assert [tuple(t.shape) for t in (kv, cu, slots, pos, count)] == [(2,), (3,), (7,), (7,), (1,)]
    assert all(t.is_contiguous() and t.is_cuda and not t.requires_grad
               for t in (kv, cu, slots, pos, count))
    want = [112, 113, 114, 111, 128, -1, -1]
    assert slots.tolist() == want and slots[2:].clone().tolist() == want[2:]
    assert pos.view(7, 1).squeeze(1).tolist() == [0, 1, 2, 15, 16, 0, 0]
    pos.fill_(5)
    kv.add_(cu[1:])
    del slots
    torch.empty(1 << 20, device=cuda_device).fill_(1.0)
    assert pos.tolist() == [5] * 7
    assert kv.tolist() == [6, 22] and cu.tolist() == [0, 3, 5] and count.tolist() == [1]
    assert torch.cat([kv, cu]).tolist() == [6, 22, 0, 3, 5]


def test_default_status_word_is_not_part_of_a_recording(cuda_device, monkeypatch):
    """The default status word is made by the first eager call, whatever status that call was
    given: one made while recording would be zeroed by every replay, with what others had
    reported in it."""
    monkeypatch.setattr(K, "_STATUS_WORDS", {})
    monkeypatch.setattr(K, "WORKSPACES", K._Workspaces())
    c = _Case(cuda_device, [70, 9], [3, 2], 8, 2, 16)
    c.run(status=torch.zeros(1, dtype=torch.int32, device=cuda_device))
    out = torch.zeros_like(c.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out)
    word = K.attention_status(cuda_device)
    word.fill_(K.STATUS_PAGES)
    graph.replay()
    torch.cuda.synchronize()
    c.check(out)
    assert int(word.item()) == K.STATUS_PAGES
