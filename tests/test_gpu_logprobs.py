"""Log probabilities, entropies and top tokens on the GPU, against their definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from wavefront_decoding_amd import ops

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def _logits(gpu, n, V, dtype=torch.float32, std=2.5, seed=0, masked=True):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(n, V, generator=g) * std
    if masked and V > 8:
        l[::3, V // 4: V // 2] = -math.inf
    return l.to(dtype).to(gpu)


def _reference(l):
    """(log p, entropy, bounds of each) of rows l in 64 bits. With d = l - max
    and Z = sum e^d: e^d is off by (|d| + 4) half steps (its argument's rounding
    and its own), the sums over V terms by at most C = 200 half steps (runs of up
    to 128 terms a thread, then a tree), so log Z by at most the mean of |d| under
    p plus C + 4, log p by 2 |d| more, and sum e d / Z by each term's."""
    l = l.double()
    d = l - l.amax(-1, keepdim=True)
    e = d.exp()
    # Z - 1 without one of the largest: next to 1, Z in 64 bits has lost it too (1.4e-13 to three digits)
    z1 = e.scatter(-1, d.argmax(-1, keepdim=True), 0.0).sum(-1, keepdim=True)
    Z, logz = 1 + z1, z1.log1p()
    lp = d - logz
    ed = torch.where(e > 0, e * d, 0.0)
    edd = torch.where(e > 0, e * d * d, 0.0)
    ent = logz - ed.sum(-1, keepdim=True) / Z
    mean, sq, C = -ed.sum(-1, keepdim=True) / Z, edd.sum(-1, keepdim=True) / Z, 200
    # z1 / Z: what of log Z comes from sums; the largest term is exact
    b_logz = EPS * ((mean + C + 4) * z1 / Z + 4 * logz)
    b_ent = 2 * b_logz + EPS * (sq + (2 * C + 16) * mean) + EPS * 4 * ent
    b_lp = b_logz + EPS * (2 * d.abs().nan_to_num(posinf=0.0) + 2 * lp.abs().nan_to_num(posinf=0.0))
    return lp, ent.squeeze(1), b_lp, b_ent.squeeze(1)


def _check(l, ids, top, got):
    out, ent, tv, ti = got
    lp, e, b_lp, b_e = _reference(l)
    rows = torch.arange(l.shape[0], device=l.device)

    def near(a, b, tol):
        same = (a.double() == b) | ((a.double() - b).abs() <= tol)
        assert same.all(), ((a.double() - b).abs() / tol).nan_to_num().max()

    if ids is not None:
        near(out, lp[rows, ids], b_lp[rows, ids])
    if ent is not None:
        near(ent, e, b_e)
    if top:
        order = torch.sort(l.float(), dim=-1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(ti, order)
        near(tv, lp.gather(1, order), b_lp.gather(1, order))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 64, 65, 255, 1000, 4096, 4099, 32000, 32768, 32769, 50257, 65536, 128000,
                               151937])
def test_sizes(gpu, dtype, V):
    n = 5
    l = _logits(gpu, n, V, dtype, seed=V)
    ids = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(V)).to(gpu)
    top = min(V, 20)
    _check(l, ids, top, ops.logprobs(l, ids, top=top, entropy=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V", [(1, 32000), (3, 200000), (300, 5000), (2050, 1001), (700, 32000)])
@pytest.mark.parametrize("top", [0, 1, 64])
def test_rows_and_tops(gpu, dtype, n, V, top):
    l = _logits(gpu, n, V, dtype, seed=n)
    ids = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(n)).to(gpu)
    _check(l, ids, top, ops.logprobs(l, ids, top=top, entropy=True))


def test_what_is_not_asked_for_is_none(gpu):
    l = _logits(gpu, 4, 500)
    ids = torch.arange(4, device=gpu)
    both = ops.logprobs(l, ids, top=3, entropy=True)
    a = ops.logprobs(l, ids)
    assert a[1:] == (None, None, None) and torch.equal(a[0], both[0])
    b = ops.logprobs(l, entropy=True)
    assert b[0] is None and b[2:] == (None, None) and torch.equal(b[1], both[1])
    c = ops.logprobs(l, top=3)
    assert c[:2] == (None, None) and torch.equal(c[2], both[2]) and torch.equal(c[3], both[3])
    assert ops.logprobs(l) == (None, None, None, None)
    assert ops.logprobs(l[:0], ids[:0], top=2)[3].shape == (0, 2)
    assert torch.equal(ops.logprobs(l, ids, n=2)[0], a[0][:2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1000, 33000])
def test_ties(gpu, dtype, V):
    """Equal logits in index order: all of them, and a few values over and over."""
    flat = torch.full((2, V), -3.5, dtype=dtype, device=gpu)
    few = torch.randint(0, 4, (6, V), generator=torch.Generator().manual_seed(V)).to(dtype).to(gpu)
    few[0, 5:] = -0.0
    few[0, :5] = 0.0
    for l in (flat, few):
        ids = torch.full((l.shape[0],), V - 1, device=gpu)
        _check(l, ids, 64, ops.logprobs(l, ids, top=64, entropy=True))


def test_confident_rows_keep_their_digits(gpu):
    """A probability next to 1: log p is what the other tokens weigh."""
    V = 32000
    for gap in (1.0, 10.0, 20.0, 40.0, 80.0):
        l = torch.zeros(2, V, device=gpu)
        l[0, 77] = gap
        l[1, V - 1] = gap
        ids = torch.tensor([77, V - 1], device=gpu)
        got = ops.logprobs(l, ids, top=2, entropy=True)
        _check(l, ids, 2, got)
        want = -math.log1p((V - 1) * math.exp(-gap))
        assert (got[0].double() - want).abs().max() <= 1e-4 * abs(want)


@pytest.mark.parametrize("V", [900, 40000])
def test_rows_that_are_not_numbers(gpu, V):
    """-inf has log p -inf; NaN, +inf and rows of -inf alone have NaN, and no other row of theirs."""
    for dtype in DTYPES:
        l = _logits(gpu, 9, V, dtype, seed=3, masked=False)
        ref = ops.logprobs(l, torch.full((9,), 5, device=gpu), top=4, entropy=True)
        bad = l.clone()
        bad[1, 700] = math.nan
        bad[1, 33] = math.nan
        bad[3, 20] = math.inf
        bad[3, 11] = math.inf
        bad[5] = -math.inf
        bad[7, 1:] = -math.inf
        bad[7, 0] = 1e30
        ids = torch.full((9,), 5, device=gpu)
        out, ent, tv, ti = ops.logprobs(bad, ids, top=4, entropy=True)
        for r in (1, 3, 5):
            assert out[r].isnan() and ent[r].isnan() and tv[r].isnan().all()
        assert ti[1, :2].tolist() == [33, 700] and ti[3, :2].tolist() == [11, 20] and ti[5].tolist() == [0, 1, 2, 3]
        assert out[7] == -math.inf and ent[7] == 0 and tv[7, 0] == 0 and ti[7].tolist() == [0, 1, 2, 3]
        assert (tv[7, 1:] == -math.inf).all()
        for r in (0, 2, 4, 6, 8):
            assert out[r] == ref[0][r] and ent[r] == ref[1][r] and torch.equal(tv[r], ref[2][r])
            assert torch.equal(ti[r], ref[3][r])


def test_huge_logits(gpu):
    l = torch.zeros(3, 2000, device=gpu)
    l[0, 3], l[0, 9] = 3e38, -3e38
    l[1] = -3e38
    l[2, :2] = 3e38
    ids = torch.tensor([9, 4, 1], device=gpu)
    out, ent, tv, ti = ops.logprobs(l, ids, top=2, entropy=True)
    assert out[0] == -math.inf and ent[0] == 0 and tv[0, 0] == 0
    assert tv[0, 1] == torch.tensor(-3e38) and ti[0].tolist() == [3, 0]
    assert abs(out[1].item() + math.log(2000)) < 1e-6 and abs(ent[1].item() - math.log(2000)) < 1e-5
    assert abs(out[2].item() + math.log(2)) < 1e-7 and ti[2].tolist() == [0, 1]


@pytest.mark.parametrize("step", [1e-45, 1e-40, 1e-38, 1e-30])
def test_logits_next_to_the_largest(gpu, step):
    """Differences too small for a float32 product: those tokens are as probable as the largest."""
    V = 600
    l = torch.zeros(4, V, device=gpu)
    l[1, 7] = l[2, 300] = step
    l[2, 11] = -step
    l[3] = -30.0
    l[3, 5], l[3, 6] = 0.0, -step
    ids = torch.tensor([0, 7, 11, 6], device=gpu)
    got = ops.logprobs(l, ids, top=3, entropy=True)
    _check(l, ids, 3, got)
    assert (got[1][:3] - math.log(V)).abs().max() < 1e-5 and abs(got[0][3].item() + math.log(2)) < 1e-6


def test_ids_outside_the_vocabulary(gpu):
    l = _logits(gpu, 5, 1000, masked=False)
    out = ops.logprobs(l, torch.tensor([-1, 1000, 999, -(2 ** 62), 2 ** 40], device=gpu))[0]
    assert out[2].isfinite() and out[[0, 1, 3, 4]].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(gpu, dtype):
    """Rows of any pitch and alignment, among them columns cut out of wider rows: the same bits as packed rows."""
    for V in (1000, 33001):
        wide = _logits(gpu, 6, V + 7, dtype, masked=False)
        ids = torch.randint(0, V, (6,), generator=torch.Generator().manual_seed(1)).to(gpu)
        for first in (0, 1, 3, 4, 7):
            cut = wide[:, first: first + V]
            got, ref = (ops.logprobs(x, ids, top=9, entropy=True) for x in (cut, cut.contiguous()))
            _check(cut, ids, 9, got)
            assert all(torch.equal(a, b) for a, b in zip(got, ref)), first
        got = ops.logprobs(wide[::2, :V], ids[:3], top=9, entropy=True)
        assert torch.equal(got[0], ops.logprobs(wide[::2, :V].contiguous(), ids[:3])[0])


def test_a_row_alone_has_the_same_bits(gpu):
    for V in (777, 32000, 100000):
        l = _logits(gpu, 40, V, seed=V)
        ids = torch.arange(40, device=gpu)
        many = ops.logprobs(l, ids, top=5, entropy=True)
        for r in (0, 1, 17, 39):
            one = ops.logprobs(l[r: r + 1], ids[r: r + 1], top=5, entropy=True)
            assert all(torch.equal(a[0], b[r]) for a, b in zip(one, many)), (V, r)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [2064385, 2097172])
def test_last_slab_shorter_than_the_top(gpu, dtype, V):
    """Vocabularies whose last slab of 32768 has 1 or 20 logits: the tokens come from logits alone, whatever the
    workspace held, also where the row is searched one token after the other."""
    l = _logits(gpu, 4, V, dtype, seed=7, masked=False)
    l[0, V - 1] = 60.0
    l[1, V - 1] = math.nan
    l[2, 5] = math.nan
    l[3] = -math.inf
    top = 64
    need = ops.logprobs_workspace_bytes(4, V, top)
    for fill in (0xff, 0x7f):
        ws = torch.full((need,), fill, dtype=torch.uint8, device=gpu)
        _, _, tv, ti = ops.logprobs(l, top=top, workspace=ws)
        for r in range(4):
            x = l[r].float()
            order = torch.sort(torch.where(x.isnan(), math.inf, x), descending=True, stable=True)[1][:top]
            assert torch.equal(ti[r], order), (fill, r)
        assert tv[0].isfinite().all() and tv[1:].isnan().all()


def test_far_rows(gpu):
    """Rows past 2^31 logits of the tensor."""
    V = 128000
    l = torch.zeros(17000, V, dtype=torch.bfloat16, device=gpu)
    l[16999, 5] = 4.0
    out, _, tv, ti = ops.logprobs(l, torch.full((17000,), 5, device=gpu), top=1)
    assert ti[16999, 0] == 5 and (ti[:16999] == 0).all()
    assert abs(out[16999].item() - (4 - math.log(V - 1 + math.exp(4)))) < 1e-5
    assert (out[:16999] + math.log(V)).abs().max() < 1e-4


def test_a_graph_replays(gpu):
    l = _logits(gpu, 12, 50000)
    ids = torch.arange(12, device=gpu)
    kw = dict(out=torch.empty(12, device=gpu), entropy_out=torch.empty(12, device=gpu),
              top_out=torch.empty(12, 6, device=gpu), top_ids=torch.empty(12, 6, dtype=torch.int64, device=gpu))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.logprobs(l, ids, top=6, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.logprobs(l, ids, top=6, **kw)
    for step in range(4):
        l.copy_(_logits(gpu, 12, 50000, seed=10 + step))
        graph.replay()
        torch.cuda.synchronize()
        ref = ops.logprobs(l, ids, top=6, entropy=True)
        assert all(torch.equal(a, b) for a, b in zip(ref, kw.values()))
