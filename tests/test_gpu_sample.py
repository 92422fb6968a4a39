"""Drawing tokens on the GPU: every id equal to the definition's, evaluated in 64 bits on the host."""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from wavefront_decoding_amd import ops

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan
LAST = 1.0 - 2.0 ** -24


def ref_one(l, u, t=1.0, k=0, p=1.0, m=0.0) -> int:
    """The definition for one row of float32 logits: weights in multiples of 2^-44 of the largest."""
    l = np.asarray(l, dtype=np.float32).astype(np.float64)
    if np.isnan(l).any():
        return int(np.isnan(l).argmax())
    if l.max() == -INF or not t > 0:
        return int(l.argmax())
    order = np.lexsort((np.arange(l.size), -l))
    with np.errstate(invalid="ignore"):
        w = np.exp((l - l.max()) / t)
    w[l == l.max()] = 1.0
    w = np.where(w > 0, np.rint(w * 2.0 ** 44) / 2.0 ** 44, 0.0)
    if 0 < k < l.size:
        order = order[:k]
    if p < 1:
        cum = np.cumsum(w[order])
        order = order[: max(1, int((cum < max(p, 0.0) * cum[-1]).sum()) + 1)]
    if m > 0:
        order = order[: max(1, int((w[order] >= m).sum()))] if m <= 1 else order[w[order] == 1.0]
    kept = np.sort(order)
    cum = np.cumsum(w[kept])
    u = min(max(u, 0.0), LAST) if u == u else 0.0
    return int(kept[int((cum <= u * cum[-1]).sum())])


def draw(gpu, logits, u, **kw):
    dev = {k: None if v is None else torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32, device=gpu)
           for k, v in kw.items()}
    return ops.sample(logits.to(gpu), torch.tensor(u, dtype=torch.float32, device=gpu), **dev).tolist()


def f32(x):
    return float(np.float32(x))


def check(gpu, logits, u, t=None, k=None, p=None, m=None):
    got = draw(gpu, logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    rows = logits.numpy()
    want = [ref_one(rows[i], f32(u[i]), f32(t[i]) if t else 1.0, k[i] if k else 0, f32(p[i]) if p else 1.0,
                    f32(m[i]) if m else 0.0) for i in range(len(u))]
    assert got == want


@pytest.mark.parametrize("V", [1, 2, 5, 63, 64, 257, 1000, 4096, 4097, 8192, 8193, 32000, 32768, 32769, 50001, 131072])
@pytest.mark.parametrize("std", [0.5, 3.0])
def test_random_rows(gpu, V, std):
    n = 24
    g = torch.Generator().manual_seed(V)
    r = lambda: torch.rand(n, generator=g)  # noqa: E731
    logits = torch.randn(n, V, generator=g) * std
    u, t, p, m = r().tolist(), (0.3 + 1.5 * r()).tolist(), (0.05 + 0.95 * r()).tolist(), (0.2 * r()).tolist()
    k = torch.randint(1, V + 3, (n,), generator=g).tolist()
    k = [x if i % 2 else min(x, 50) for i, x in enumerate(k)]
    check(gpu, logits, u)
    check(gpu, logits, u, t)
    check(gpu, logits, u, t, k)
    check(gpu, logits, u, t, p=p)
    check(gpu, logits, u, t, m=m)
    check(gpu, logits, u, t, k, p)
    mix = lambda x, off, s: [off if (i >> s) % 2 else v for i, v in enumerate(x)]  # noqa: E731
    check(gpu, logits, u, mix(t, 0.0, 3), mix(k, 0, 0), mix(p, 1.0, 1), mix(m, 0.0, 2))


@pytest.mark.parametrize("V", [16, 300, 5000, 40000])
def test_equal_logits(gpu, V):
    """Few distinct values: the limits cut inside runs of equals, lowest indexes first;
    u and the sums are exact, so a draw on a border has one answer."""
    n = 40
    g = torch.Generator().manual_seed(V)
    logits = torch.randint(0, 3, (n, V), generator=g).float() * 0.0
    logits[n // 2:] = torch.randint(0, 4, (n - n // 2, V), generator=g).float() * 200.0  # lower ones weigh nothing
    logits[3, ::2] = -0.0  # the same value
    u = [(i % 16) / 16 for i in range(n)]
    k = [1 + (7 * i) % V for i in range(n)]
    p = [(i % 8) / 8 for i in range(n)]
    check(gpu, logits, u)
    check(gpu, logits, u, k=k)
    check(gpu, logits, u, p=p)
    check(gpu, logits, u, k=k, p=p)
    check(gpu, logits, u, k=k, p=p, m=[1.0] * n)
    flat = torch.zeros(16, 16)
    assert draw(gpu, flat, [j / 16 for j in range(16)]) == list(range(16))


def test_bf16_logits_with_many_ties(gpu):
    n, V = 32, 32000
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(n, V, generator=g).bfloat16().float() * 2
    u, p = torch.rand(n, generator=g).tolist(), torch.rand(n, generator=g).tolist()
    k = torch.randint(1, 3000, (n,), generator=g).tolist()
    check(gpu, logits, u, k=k)
    check(gpu, logits, u, p=p)
    check(gpu, logits, u, [0.7] * n, k, p)


@pytest.mark.parametrize("V", [3000, 20000, 60000])
def test_every_top_k_over_few_values(gpu, V):
    """Every k around and between the ends of the runs of equal logits, to past a sorted list."""
    g = torch.Generator().manual_seed(V)
    row = (torch.randn(V, generator=g) * 2).bfloat16().float()
    ends = torch.unique(row, return_counts=True)[1].flip(0).cumsum(0)
    ends = ends[ends < 2500][::3].tolist()
    k = sorted({e + d for e in ends for d in (-1, 0, 1) if e + d > 0})
    rows = row.expand(len(k), V).contiguous()
    check(gpu, rows, torch.rand(len(k), generator=g).tolist(), k=k)
    check(gpu, rows, torch.rand(len(k), generator=g).tolist(), k=k, p=[0.9] * len(k))


@pytest.mark.parametrize("V", [70, 9000, 33000])
def test_masked_and_special_logits(gpu, V):
    g = torch.Generator().manual_seed(V)
    rows = torch.randn(12, V, generator=g)
    rows[0] = -INF                       # nothing left
    rows[1] = -INF
    rows[1, V - 1] = 0.5                 # one token left, the last
    rows[2, : V - 3] = -INF              # three left
    rows[3, : V - 3] = torch.finfo(torch.float32).min  # masked by the type's lowest value
    rows[4] = torch.finfo(torch.float32).min           # all at the lowest value: equals
    rows[5, V // 2] = NAN
    rows[6, [3, V // 2, V - 2]] = INF    # shared by three
    rows[7, V // 3] = INF
    rows[8] = 3.4e38
    rows[8, ::2] = -3.4e38
    rows[9, 5:] = -INF
    rows[10, ::2] = -INF
    for u in (0.0, 0.4, 0.7, LAST):
        us = [u] * 12
        check(gpu, rows, us)
        check(gpu, rows, us, t=[0.8] * 12, k=[4] * 12)
        check(gpu, rows, us, t=[1.3] * 12, p=[0.6] * 12)
        check(gpu, rows, us, p=[0.9] * 12, m=[0.3] * 12, k=[5] * 12)


@pytest.mark.parametrize("V", [3000, 30000, 100000])
@pytest.mark.parametrize("masked", [-INF, -1e9, -1e4])
def test_whole_stretches_masked(gpu, V, masked):
    """A grammar leaves a few tokens, far apart, of a row; fewer than top-k, or many."""
    n = 24
    g = torch.Generator().manual_seed(V)
    rows = torch.randn(n, V, generator=g) * 2
    for i in range(n):
        left = [1, 3, 40, 900][i % 4]
        keep = torch.randperm(V, generator=g)[:left] if i % 8 < 4 else torch.arange(V - left, V)
        mask = torch.ones(V, dtype=torch.bool)
        mask[keep] = False
        rows[i, mask] = masked
    u = torch.rand(n, generator=g).tolist()
    for k in (5, 100, 500, 2000):
        check(gpu, rows, u, k=[k] * n)
        check(gpu, rows, u, [1.3] * n, [k] * n, [0.9] * n)
    check(gpu, rows, u, p=[0.95] * n)
    check(gpu, rows, u, [0.7] * n, m=[0.02] * n)


def test_parameters_outside_their_ranges(gpu):
    V = 500
    l = torch.randn(1, V, generator=torch.Generator().manual_seed(2))
    cases = [dict(t=x) for x in (0.0, -1.0, NAN, INF, 1e-30, 1e30, 1e-45)]
    cases += [dict(k=x) for x in (0, -5, V, V + 1, 2 ** 31 - 1, 1)]
    cases += [dict(p=x) for x in (0.0, -1.0, 1.0, 2.0, NAN, 1e-30, LAST)] + [dict(m=x) for x in (0.0, -1.0, 1.0, 2.0, NAN)]
    for u in (0.0, 0.5, 0.999, 1.0, 7.0, -3.0, NAN):
        rows = l.expand(len(cases), V).contiguous()
        kw = {n: [c.get(s, d) for c in cases] for n, s, d in (("t", "t", 1.0), ("k", "k", 0), ("p", "p", 1.0),
                                                             ("m", "m", 0.0))}
        got = draw(gpu, rows, [u] * len(cases), temperature=kw["t"], top_k=kw["k"], top_p=kw["p"], min_p=kw["m"])
        for c, id_ in zip(cases, got):
            t, p, m = c.get("t", 1.0), c.get("p", 1.0), c.get("m", 0.0)
            assert id_ == ref_one(l[0].numpy(), f32(u), f32(t), c.get("k", 0), 1.0 if p != p else f32(p),
                                  0.0 if m != m else f32(m)), (c, u)


def test_draws_follow_the_distribution(gpu):
    """u at the middles of N equal steps: a token is drawn p N times, give or take one."""
    N, V = 4096, 50
    l = torch.randn(1, V, generator=torch.Generator().manual_seed(3)) * 1.5
    ids = ops.sample(l.expand(N, V).contiguous().to(gpu), ((torch.arange(N) + 0.5) / N).to(gpu))
    count = torch.bincount(ids.cpu(), minlength=V).double()
    assert (count - N * torch.softmax(l[0].double(), 0)).abs().max() <= 1.0


def test_row_pitches_and_alignment(gpu):
    g = torch.Generator().manual_seed(4)
    for V, pitch, off in ((1001, 1001, 0), (1001, 1003, 1), (8190, 8191, 3), (33001, 33001, 0)):
        big = torch.randn(9 * pitch + off, generator=g)
        view = big[off:].as_strided((9, V), (pitch, 1))
        u = torch.rand(9, generator=g).tolist()
        want = [ref_one(view[i].numpy(), f32(u[i]), k=40, p=f32(0.8)) for i in range(9)]
        dev = big.to(gpu)[off:].as_strided((9, V), (pitch, 1))
        got = ops.sample(dev, torch.tensor(u, device=gpu), top_k=torch.full((9,), 40, dtype=torch.int32, device=gpu),
                         top_p=torch.full((9,), 0.8, device=gpu))
        assert got.tolist() == want


def test_a_row_does_not_see_its_companions(gpu):
    n, V = 64, 32000
    g = torch.Generator().manual_seed(5)
    l, u = (torch.randn(n, V, generator=g) * 2).to(gpu), torch.rand(n, generator=g).to(gpu)
    p = torch.full((n,), 0.9, device=gpu)
    ids = ops.sample(l, u, top_p=p)
    assert torch.equal(ops.sample(l, u, top_p=p), ids)
    for i in (0, 17, 63):
        assert ops.sample(l[i: i + 1], u[i: i + 1], top_p=p[:1]).item() == ids[i].item()


def test_ring_and_accept_flags(gpu):
    n, V = 6, 900
    g = torch.Generator().manual_seed(6)
    l, u = torch.randn(n, V, generator=g).to(gpu), torch.rand(n, generator=g).to(gpu)
    ids = ops.sample(l, u)
    ring = torch.full((8,), -7, dtype=torch.int64, device=gpu)
    ring[7] = ids[2]
    rows = torch.tensor([4, 0, -1, 3, 8, 1], dtype=torch.int32, device=gpu)  # -1 and 8: nowhere
    expect = torch.stack([ids[0], ids[1] + 1, torch.tensor(-8, device=gpu), ids[3], torch.tensor(-99, device=gpu),
                          ids[5]])
    accept = torch.full((n,), -1, dtype=torch.int32, device=gpu)
    out = torch.full((n + 2,), -5, dtype=torch.int64, device=gpu)
    got = ops.sample(l, u, n=n, out=out, ring=ring, ring_rows=rows, expect=expect, accept=accept)
    assert got is out and torch.equal(out[:n], ids) and out[n:].tolist() == [-5, -5]
    assert accept.tolist() == [1, 0, 1, 1, 0, 1]
    want = [-7] * 7 + [ids[2].item()]
    for r, i in zip(rows.tolist(), ids.tolist()):
        if 0 <= r < 8:
            want[r] = i
    assert ring.tolist() == want


def test_captured_draw(gpu):
    n, V = 5, 32000
    g = torch.Generator().manual_seed(7)
    l, u = torch.randn(n, V, device=gpu), torch.rand(n, device=gpu)
    p, k = torch.full((n,), 0.9, device=gpu), torch.full((n,), 300, dtype=torch.int32, device=gpu)
    ops.sample(l, u, top_p=p, top_k=k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample(l, u, top_p=p, top_k=k)
    for _ in range(4):
        l.copy_(torch.randn(n, V, generator=g) * 2)
        u.copy_(torch.rand(n, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.sample(l, u, top_p=p, top_k=k))
    assert ops.sample(l[:0], u[:0]).numel() == 0


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.7, top_k=40, top_p=0.9), dict(temperature=0.0),
                                dict(temperature=1.5, min_p=0.05)])
def test_sampled_wavefront_is_sequential_sampling(gpu, kw):
    """Drafts and their verification draw with the position's number: WFD and
    draft-then-verify commit what sequential decoding with that seed draws."""
    from wavefront_decoding_amd import model as M
    from wavefront_decoding_amd.acceptance import SeededSampler
    from wavefront_decoding_amd.blocks import LoopedBlocks
    from wavefront_decoding_amd.engine import LoopedModel
    from wavefront_decoding_amd.policy import SampledPolicy
    from wavefront_decoding_amd.scheduler import generate_draft_then_verify, generate_wavefront_dynamic

    cfg = M.CONFIGS["tiny"]
    blocks = LoopedBlocks(LoopedModel(cfg, M.init_weights(cfg, 0), gpu, max_seq_len=64))
    ids = torch.randint(0, cfg.vocab_size, (20,), generator=torch.Generator().manual_seed(0)).to(gpu)
    runs = []
    for seed in (0, 1):
        want, _ = blocks.ar_generate(ids, 16, sampler=SeededSampler(seed, **kw))
        policy = SampledPolicy(cfg.T_total, 2, sample_seed=seed, **({"temperature": 1.0} | kw))
        assert generate_wavefront_dynamic(blocks, ids, 16, policy)[0] == want
        assert generate_draft_then_verify(blocks, ids, 16, policy, 3)[0] == want
        runs.append(want)
    if kw.get("temperature") != 0.0:
        assert runs[0] != runs[1]


@pytest.mark.parametrize("V", [2000, 40000])
def test_top_p_at_the_edge_of_a_bin(gpu, V):
    """a tokens of one logit and the rest of a lower one, top-p at the first ones' share:
    whether the second ones' bin is needed is a matter of the last bit of p."""
    g = torch.Generator().manual_seed(V)
    n = 96
    logits = torch.zeros(n, V)
    t, p = [], []
    for i in range(n):
        at = torch.randperm(V, generator=g)
        a, gap = V // 3 + i, 1.0 + i / 64
        logits[i, at[a:]] = -gap
        t.append([1.0, 0.75, 1.5][i % 3])
        share = np.float32(a / (a + (V - a) * math.exp(-gap / t[-1])))
        p.append(float(np.nextafter(share, np.float32(i % 2), dtype=np.float32) if i % 4 < 2 else share))
    check(gpu, logits, torch.rand(n, generator=g).tolist(), t, None, p)
    check(gpu, logits, [LAST] * n, t, None, p)


@pytest.mark.parametrize("V", [300, 20000, 60000])
@pytest.mark.parametrize("t", [INF, 1e30, 1e-30, 1e-45])
def test_extreme_temperatures_over_masked_rows(gpu, V, t):
    g = torch.Generator().manual_seed(V)
    n = 6
    rows = torch.randn(n, V, generator=g) * 3
    rows[1, ::2] = -INF
    rows[2, : V - 7] = -INF
    rows[3, 5:] = torch.finfo(torch.float32).min
    rows[4, [1, V - 1]] = rows[4].max() + 1  # two largest
    u = torch.rand(n, generator=g).tolist()
    check(gpu, rows, u, [t] * n)
    check(gpu, rows, u, [t] * n, None, [0.6] * n)
    check(gpu, rows, u, [t] * n, [50] * n, [0.6] * n)
    check(gpu, rows, u, [t] * n, None, [0.9] * n, [0.5] * n)


@pytest.mark.parametrize("V", [5, 300, 20000, 60000])
def test_min_p_above_one_keeps_the_first_token_alone(gpu, V):
    """No weight reaches it, and only the first of the order stays whatever its weight: not
    the others as large. At 1 these stay."""
    g = torch.Generator().manual_seed(V)
    n = 8
    rows = torch.randn(n, V, generator=g).clamp(max=3.0)
    at = torch.stack([torch.randperm(V, generator=g)[:3].sort().values for _ in range(n)])
    rows.scatter_(1, at, 5.0)
    rows[5].scatter_(0, at[5], INF)
    rows[6] = -INF
    rows[7] = 0.0
    first = at[:, 0].tolist()
    first[6] = first[7] = 0
    for u in (0.0, 0.5, LAST):
        us = [u] * n
        for kw in (dict(), dict(top_p=[0.9] * n), dict(top_k=[4] * n), dict(top_k=[50] * n, top_p=[0.9] * n)):
            for m in (1.0000001, 2.0, INF):
                assert draw(gpu, rows, us, min_p=[m] * n, **kw) == first
            if not kw:
                last = draw(gpu, rows, us, min_p=[1.0] * n)
                assert last[:6] == [int(a[min(2, int(u * 3))]) for a in at[:6]]


def ref_int(l, u, t=1.0, k=0, p=1.0) -> int:
    """The definition with its weights as integers, multiples of 2^-44 of the largest, and every
    sum and product exact."""
    l = np.asarray(l, dtype=np.float32).astype(np.float64)
    w = np.rint(np.exp((l - l.max()) / t) * 2.0 ** 44).astype(np.uint64)
    order = np.lexsort((np.arange(l.size), -l))
    if 0 < k < l.size:
        order = order[:k]
    if p < 1:
        cum = np.cumsum(w[order], dtype=np.uint64)  # at most 2^63
        need = math.ceil(Fraction(p) * int(cum[-1]))
        order = order[: int(np.searchsorted(cum, np.uint64(max(need, 1)), side="left")) + 1]
    kept = np.sort(order)
    cum = np.cumsum(w[kept], dtype=np.uint64)
    return int(kept[np.searchsorted(cum, np.uint64(math.floor(Fraction(u) * int(cum[-1]))), side="right")])


@pytest.mark.parametrize("V", [1 << 19, (1 << 19) - 1, (1 << 19) - 8191])
def test_largest_vocabularies_flat(gpu, V):
    """Weights of one, whose sum reaches 2^63 and a thread's 2^53; the list overflows, so the row
    is drawn by one workgroup with top-p, and with a top-k past the lists'."""
    us = [0.0, 2.0 ** -24, 0.25, 0.7, LAST]
    flat = torch.zeros(len(us), V)
    token = lambda n: [math.floor(Fraction(f32(u)) * n) for u in us]  # noqa: E731
    assert draw(gpu, flat, us) == token(V)
    for k in (1, 600, 601, 5000, V - 1):
        assert draw(gpu, flat, us, top_k=[k] * len(us)) == token(k)
    for p in (2.0 ** -30, 0.3, LAST):
        kept = max(1, math.ceil(Fraction(f32(p)) * V))
        assert draw(gpu, flat, us, top_p=[p] * len(us)) == token(kept)
        kept = math.ceil(Fraction(f32(p)) * 5000)
        assert draw(gpu, flat, us, top_p=[p] * len(us), top_k=[5000] * len(us)) == token(kept)


@pytest.mark.parametrize("V", [1 << 19, (1 << 19) - 1])
@pytest.mark.parametrize("std", [0.2, 2.0])
def test_largest_vocabularies_random(gpu, V, std):
    g = torch.Generator().manual_seed(V)
    n = 4
    rows = torch.randn(n, V, generator=g) * std
    t = [1.0, 0.7, 1.3, 0.5]
    host = rows.numpy()
    for k, p in ((0, 1.0), (0, 0.9), (0, 0.3), (40, 1.0), (300, 0.95), (600, 1.0), (601, 1.0), (601, 0.9),
                 (20000, 0.5), (300000, 0.99)):
        for u in (torch.rand(n, generator=g).tolist(), [LAST] * n):
            got = draw(gpu, rows, u, temperature=t, top_k=[k] * n, top_p=[p] * n)
            assert got == [ref_int(host[i], f32(u[i]), f32(t[i]), k, f32(p)) for i in range(n)], (k, p, u)
