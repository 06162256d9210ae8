"""ddt_sample against a plain implementation in whole numbers (exact tokens) and in 64-bit
floating point (log-probabilities), and its distribution.  Replaces sample() at temperature > 0
(model/utils.py:28-35)."""
import math

import numpy as np
import pytest
import torch

import inputs as gin
from mdflash_b200 import _lib
from mdflash_b200 import kernels as K

pytestmark = pytest.mark.gpu


def _reference(x, u, temp, top_k, top_p, min_p, exp):
    """One row on the host (numpy): the definition, token by token in sorted order.  `exp`: the
    float32 exponentials of this row (their values define the weights)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float32))
    V = x.size
    top = x.max()
    if top == -np.inf:
        return -1, -math.inf
    order = np.lexsort((np.arange(V), -x))
    if temp < 1e-5:
        return int(order[0]), 0.0
    w = (exp.astype(np.float64) * 2.0 ** 40).astype(np.int64).astype(object)
    k = top_k if 0 < top_k < V else V
    kept = order[:k]
    if top_p < 1.0:
        reach = np.float64(np.float32(top_p)) * np.float64(int(sum(w[kept])))
        before, n = 0, 0
        for i in kept:
            if n > 0 and not np.float64(int(before)) < reach:
                break
            before += w[i]
            n += 1
        kept = kept[:n]
    kept = np.sort([i for i in kept if exp[i] >= np.float32(min(min_p, 1.0))])
    total = int(sum(w[kept]))
    target = int(math.floor(np.float64(np.float32(u)) * np.float64(total)))
    target = max(min(target, total - 1), 0)
    run = 0
    for i in kept:
        run += int(w[i])
        if run > target:
            break
    z = 0.0 if x[i] == top else (float(x[i]) - float(top)) / float(np.float32(temp))
    return int(i), z - (math.log(total) - 40 * math.log(2.0))


def _check(dev, x, u, temp, k=None, p=None, mp=None):
    rows = x.shape[0]
    to = lambda v, dt: None if v is None else torch.tensor(v, dtype=dt, device=dev)  # noqa: E731
    args = (to(temp, torch.float32), to(k, torch.int32), to(p, torch.float32), to(mp, torch.float32))
    tok, logp = K.sample(x, to(u, torch.float32), *args)
    xf = torch.where(torch.isnan(x), -math.inf, x.float())
    top = xf.amax(-1, keepdim=True)
    t = torch.where(args[0] < 1e-5, 1.0, args[0])[:, None]
    exp = torch.exp(torch.where(xf == top, 0.0, (xf - top) / t)).cpu().numpy()
    xh = x.float().cpu().numpy()
    for r in range(rows):
        want, lp = _reference(xh[r], u[r], temp[r], k[r] if k else 0, p[r] if p else 1.0,
                              mp[r] if mp else 0.0, exp[r])
        assert int(tok[r]) == want, (r, int(tok[r]), want)
        # one rounding of z to fp32 and one of the result
        got = float(logp[r])
        assert got == lp or abs(got - lp) <= 2.0 ** -22 * (abs(lp) + abs(math.log(1 + x.shape[1]))), \
            (r, got, lp)
    return tok, logp


def _rules(rng, rows):
    return ([float(v) for v in rng.choice([0.0, 0.3, 0.7, 1.0, 1.7], rows)],
            [int(v) for v in rng.choice([0, 1, 2, 17, 50, 1000], rows)],
            [float(v) for v in rng.choice([1.0, 0.0, 0.01, 0.5, 0.9, 0.999], rows)],
            [float(v) for v in rng.choice([0.0, 0.02, 0.3, 1.0, 2.0], rows)])


@pytest.mark.parametrize("V", [1, 2, 7, 31, 33, 255, 1000, 1025, 4097, 20000, 40961])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_matches_definition(cuda_device, V, dtype):
    rng = np.random.default_rng(V)
    rows = 24 if V < 5000 else 8
    x = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 3).to(dtype)
    u = [float(np.float32(v)) for v in rng.random(rows)]
    u[0] = 0.0
    u[1] = float(np.nextafter(np.float32(1), np.float32(0)))
    _check(cuda_device, x.to(cuda_device), u, *_rules(rng, rows))


@pytest.mark.parametrize("only", ["temperature", "k", "p", "min_p"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_full_vocabulary(cuda_device, only, dtype):
    rng = np.random.default_rng(len(only))
    rows = 6
    x = torch.from_numpy(rng.standard_normal((rows, gin.V_QWEN3)).astype(np.float32) * 2).to(dtype)
    u = [float(np.float32(v)) for v in rng.random(rows)]
    temp = [0.5, 0.9, 1.0, 1.3, 3.0, 20.0]
    k = [1, 5, 50, 999, 30000, 151935] if only == "k" else None
    p = [0.1, 0.5, 0.9, 0.95, 0.999, 0.99999] if only == "p" else None
    mp = [0.5, 0.1, 0.05, 0.01, 0.001, 1e-7] if only == "min_p" else None
    _check(cuda_device, x.to(cuda_device), u, temp, k, p, mp)


@pytest.mark.parametrize("p", [0.05, 0.5, 0.9, 0.95, 0.9999])
@pytest.mark.parametrize("spread,heavy", [(0.3, 0), (3.0, 0), (3.0, 8), (8.0, 3), (0.01, 0)])
def test_sample_nucleus_boundaries(cuda_device, p, spread, heavy):
    """top-p alone over rows from flat (the nucleus is most of the vocabulary) to spiky (a few
    tokens), where the boundary is first judged by intervals of the logits; temperatures whose
    quotients are awkward (significands of all ones)."""
    rng = np.random.default_rng(int(p * 1e4) + heavy)
    rows, V = 4, 60001
    x = rng.standard_normal((rows, V)).astype(np.float32) * spread
    for r in range(rows):
        x[r, rng.integers(0, V, heavy)] += rng.random(heavy).astype(np.float32) * 12
    u = [float(np.float32(v)) for v in rng.random(rows)]
    temp = [1.0, float(np.nextafter(np.float32(1), np.float32(0))), 0.7,
            float(np.nextafter(np.float32(2), np.float32(0)))]
    mp = [0.0, 0.0, 0.001, 0.2]
    for dtype in (torch.float32, torch.bfloat16):
        _check(cuda_device, torch.from_numpy(x).to(dtype).to(cuda_device), u, temp, None, [p] * rows, mp)


@pytest.mark.parametrize("k", [1200, 1300, 2047, 5000, 59999])
def test_sample_long_candidate_lists(cuda_device, k):
    """top-k around and beyond what one list holds, with and without top-p, NaN in the row."""
    rng = np.random.default_rng(k)
    rows, V = 3, 60001
    x = rng.standard_normal((rows, V)).astype(np.float32) * 2
    x[1, ::3] = np.nan
    x[2, 100:59000] = -np.inf
    u = [float(np.float32(v)) for v in rng.random(rows)]
    for p in (1.0, 0.97):
        _check(cuda_device, torch.from_numpy(x).to(cuda_device), u, [0.9] * rows, [k] * rows,
               [p] * rows, [0.0] * rows)


def test_sample_ties(cuda_device):
    """Rows of a few distinct values: cuts fall inside long runs of equal logits, which are
    kept from the lowest index."""
    rng = np.random.default_rng(5)
    rows, V = 40, 3001
    x = torch.from_numpy(rng.choice([0.0, -0.0, 1.0, -2.0], (rows, V)).astype(np.float32))
    x[0] = 0.0
    x[1] = -0.0
    u = [float(np.float32(v)) for v in rng.random(rows)]
    temp, k, p, mp = _rules(rng, rows)
    k = [int(v) for v in rng.integers(0, V + 2, rows)]
    p = [float(np.float32(v)) for v in rng.random(rows)]
    _check(cuda_device, x.to(cuda_device), u, temp, k, p, mp)
    _check(cuda_device, x.to(torch.bfloat16).to(cuda_device), u, temp, k, p, [0.0] * rows)


def test_sample_masked_and_odd_values(cuda_device):
    """-inf and NaN are never drawn, +inf takes all, the type's lowest value is a value, rows
    without anything to draw give -1 and -inf."""
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    V = 70
    base = torch.randn((9, V), generator=torch.Generator().manual_seed(1))
    base[0] = -inf
    base[1] = nan
    base[2] = nan
    base[2, 5] = -inf
    base[3] = -inf
    base[3, 69] = -3.0
    base[4, ::2] = nan
    base[4, 1::4] = -inf
    base[5, 40] = inf
    base[5, 41] = inf
    base[5, 0] = nan
    base[6] = low
    base[7] = low
    base[7, 3] = 0.0
    base[8, :50] = -inf
    for temp in (0.0, 1.0, 0.5):
        for k, p in ((0, 1.0), (3, 1.0), (0, 0.8), (60, 0.99)):
            for u in (0.0, 0.37, 0.999):
                tok, logp = _check(cuda_device, base.to(cuda_device), [u] * 9, [temp] * 9, [k] * 9,
                                   [p] * 9, [0.0] * 9)
                t = tok.tolist()
                assert t[:4] == [-1, -1, -1, 69] and t[5] in (40, 41) and t[7] == 3
                assert t[4] % 4 == 3 and t[8] >= 50 and t[6] >= 0
                assert logp[:3].tolist() == [-inf] * 3


def test_sample_does_not_depend_on_the_batch_or_strides(cuda_device):
    g = torch.Generator().manual_seed(8)
    rows, V = 37, 9001
    wide = (torch.randn((rows, V + 13), generator=g) * 3).to(cuda_device)
    x = wide[:, 5:5 + V]  # rows that start at odd addresses
    u = torch.rand(rows, generator=g).to(cuda_device)
    temp = torch.full((rows,), 0.8, device=cuda_device)
    k = torch.full((rows,), 400, dtype=torch.int32, device=cuda_device)
    p = torch.full((rows,), 0.9, device=cuda_device)
    tok, logp = K.sample(x, u, temp, k, p)
    tok2, logp2 = K.sample(x.contiguous(), u, temp, k, p)
    assert torch.equal(tok, tok2) and torch.equal(logp, logp2)
    for r in range(0, rows, 6):
        one = K.sample(x[r:r + 1], u[r:r + 1], temp[r:r + 1], k[r:r + 1], p[r:r + 1])
        assert torch.equal(one[0], tok[r:r + 1]) and torch.equal(one[1], logp[r:r + 1])


@pytest.mark.parametrize("rows", [7, 40, 100, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_full_vocabulary_at_every_launch_shape(cuda_device, rows, dtype):
    """A batch's size decides how many CTAs share a row (8, 4, 2, 1, or what keeps the rows in
    flight in L2): every row's token and log-probability are those of the row alone, whatever its
    rules, and the first rows' those of the definition."""
    g = torch.Generator(cuda_device).manual_seed(rows)
    rng = np.random.default_rng(rows)
    x = torch.empty((rows, gin.V_QWEN3), device=cuda_device).normal_(0, 3, generator=g)
    x[::3] *= 0.2
    x[1::7, ::2] = float("nan")
    x[2::7, 1000:150000] = -math.inf
    x = x.to(dtype)
    u = [float(np.float32(v)) for v in rng.random(rows)]
    temp, k, p, mp = _rules(rng, rows)
    k = [0 if r % 2 else v for r, v in enumerate(k)]  # half of the rows: top-p alone
    to = lambda v, dt=torch.float32: torch.tensor(v, dtype=dt, device=cuda_device)  # noqa: E731
    args = (to(u), to(temp), to(k, torch.int32), to(p), to(mp))
    tok, logp = K.sample(x, *args)
    alone = [K.sample(x[r:r + 1], *(a[r:r + 1] for a in args)) for r in range(rows)]
    assert torch.equal(tok, torch.cat([t for t, _ in alone]))
    assert torch.equal(logp, torch.cat([v for _, v in alone]))
    n = 4
    first = _check(cuda_device, x[:n], u[:n], temp[:n], k[:n], p[:n], mp[:n])
    assert torch.equal(first[0], tok[:n]) and torch.equal(first[1], logp[:n])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 9001, 40960])
def test_sample_several_draws_from_one_row(cuda_device, dtype, V):
    """One row of logits expanded to many (stride 0), the last row of its storage: every draw is
    the one of a copy of the row.  Rows that overlap in any other way are refused."""
    g = torch.Generator().manual_seed(V)
    rows = 37
    x = (torch.randn((3, V), generator=g) * 3).to(dtype).to(cuda_device)
    u = torch.rand(rows, generator=g).to(cuda_device)
    temp = torch.full((rows,), 0.8, device=cuda_device)
    k = torch.tensor([0, 40, 0] * 12 + [5], dtype=torch.int32, device=cuda_device)
    p = torch.tensor([1.0, 0.9, 0.8] * 12 + [1.0], device=cuda_device)
    wide = x[2].expand(rows, V)
    assert wide.stride(0) == 0
    tok, logp = K.sample(wide, u, temp, k, p)
    tok2, logp2 = K.sample(wide.contiguous(), u, temp, k, p)
    assert torch.equal(tok, tok2) and torch.equal(logp, logp2)
    one = K.sample(x[2:], u[:1], temp[:1], k[:1], p[:1])
    assert torch.equal(one[0], tok[:1]) and torch.equal(one[1], logp[:1])
    with pytest.raises(_lib.DDTreeError):
        K.sample(x.flatten().as_strided((4, V), (V // 2, 1)), u[:4], temp[:4])


@pytest.mark.parametrize("k,p,mp", [(0, 1.0, 0.0), (6, 1.0, 0.0), (0, 0.8, 0.0), (0, 1.0, 0.2)])
def test_sample_distribution(cuda_device, k, p, mp):
    """120k draws from 16 tokens: a chi-square test against the truncated softmax (at most 15
    degrees of freedom, threshold at p ~ 1e-6)."""
    g = torch.Generator().manual_seed(21)
    V, S, T = 16, 120_000, 0.9
    x = torch.randn(V, generator=g) * 2
    w = torch.softmax(x.double() / T, -1)
    order = torch.argsort(w, descending=True)
    keep = torch.zeros(V, dtype=torch.bool)
    n = k if k else V
    cum = torch.cumsum(w[order][:n] / w[order][:n].sum(), 0)
    n = min(n, int((cum - w[order][:n] / w[order][:n].sum() < p).sum())) if p < 1 else n
    keep[order[:n]] = True
    keep &= w / w.max() >= mp
    w = torch.where(keep, w, 0.0)
    w = (w / w.sum()).numpy()
    f = lambda v, dt=torch.float32: torch.full((S,), v, dtype=dt, device=cuda_device)  # noqa: E731
    tok, logp = K.sample(x.to(cuda_device).expand(S, V).contiguous(),
                         torch.rand(S, generator=g).to(cuda_device), f(T), f(k, torch.int32), f(p),
                         f(mp))
    counts = np.bincount(tok.cpu().numpy(), minlength=V)
    assert counts[w == 0].sum() == 0
    live = w > 0
    chi2 = float((((counts - w * S) ** 2)[live] / (w * S)[live]).sum())
    assert chi2 < 55.0, chi2
    np.testing.assert_allclose(np.exp(logp.cpu().double().numpy()), w[tok.cpu().numpy()], rtol=1e-5)


def test_sample_refusals(cuda_device):
    x = torch.zeros((2, 8), device=cuda_device)
    one = torch.ones(2, device=cuda_device)
    with pytest.raises(ValueError):
        K.sample(x.cpu(), one, one)
    with pytest.raises(TypeError):
        K.sample(x.half(), one, one)
    with pytest.raises(ValueError):
        K.sample(x, one[:1], one)
    with pytest.raises(ValueError):
        K.sample(x, one, one, top_k=one)
    with pytest.raises(ValueError):
        K.sample(x.t(), one, one)
    with pytest.raises(_lib.DDTreeError):
        K.sample(torch.zeros((1, 1 << 22), device=cuda_device), one[:1], one[:1])
    tok, logp = K.sample(x[:0], one[:0], one[:0])
    assert tok.shape == (0,) and logp.shape == (0,)
