"""Attention of rows that share a prefix, on the GPU, against its definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from tests.serving_ref import attend, check_attention
from wavefront_decoding_amd import ops

pytestmark = pytest.mark.gpu

P_STEP = {torch.bfloat16: 2.0 ** -16, torch.float32: 0.0}  # probabilities meet V in two bf16 terms


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class Case:
    """Caches of `rows` random rows (token-major or in blocks) and a call's tables.
    groups: (prefix base, prefix length, rows); own: (base, length) per row."""

    def __init__(self, gpu, dtype, H, Hkv, Dh, rows, groups, own, *, block=0, seed=0, lead=0, std=1.0):
        g = _gen(seed)
        self.k, self.v = (torch.randn(rows, Hkv, Dh, generator=g).to(dtype) for _ in range(2))
        n = len(own)
        self.q = (torch.randn(n, H, Dh, generator=g) * std).to(dtype)
        first = [lead]
        for _, _, c in groups:
            first.append(first[-1] + c)
        self.gpu, self.groups, self.own, self.first, self.block = gpu, groups, own, first, block
        self.dtype, self.Hkv = dtype, Hkv

    def dev(self, x, dtype):
        return torch.tensor(x, dtype=dtype, device=self.gpu)

    def layout(self, t):
        if not self.block:
            return t.to(self.gpu)
        return t.view(-1, self.block, *t.shape[1:]).transpose(1, 2).contiguous().to(self.gpu)

    def args(self, rows=None):
        """The call's positional arguments, for all rows or a choice of them (kept in their groups)."""
        rows = list(range(len(self.own))) if rows is None else rows
        first = [sum(r < f for r in rows) for f in self.first]
        return (self.q[rows].to(self.gpu), self.layout(self.k), self.layout(self.v),
                self.dev([p for p, _, _ in self.groups], torch.int64),
                self.dev([length for _, length, _ in self.groups], torch.int32), self.dev(first, torch.int32),
                self.dev([self.own[r][0] for r in rows], torch.int64),
                self.dev([self.own[r][1] for r in rows], torch.int32))

    def maxima(self):
        return dict(prefix_len_max=max([length for _, length, _ in self.groups] + [0]),
                    kv_len_max=max(length for _, length in self.own),
                    group_max=max([c for _, _, c in self.groups] + [0]))

    def run(self, rows=None, **kw):
        return ops.attn_shared(*self.args(rows), **(self.maxima() | kw))

    def keys(self, i):
        at = []
        for j, (base, length, _) in enumerate(self.groups):
            if self.first[j] <= i < self.first[j + 1]:
                at += range(base, base + max(length, 0))
        base, length = self.own[i]
        return at + list(range(base, base + max(length, 0)))

    def check(self, out, scale=None):
        scale = 1 / math.sqrt(self.q.shape[-1]) if scale is None else scale
        for i in range(len(self.own)):
            at = self.keys(i)
            ref, bound = attend(self.q[i].double(), self.k[at].double().transpose(0, 1),
                                self.v[at].double().transpose(0, 1), scale, P_STEP[self.dtype])
            check_attention(out[i], ref, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv,Dh", [(4, 4, 64), (4, 4, 128), (4, 2, 128), (8, 2, 64), (3, 1, 128), (8, 1, 64),
                                      (16, 1, 128), (16, 16, 128)])
def test_groups_of_every_size(gpu, dtype, H, Hkv, Dh):
    """Groups of 1 to 40 rows (beyond a workgroup's), ragged prefixes and own keys,
    an empty group, rows before and behind the groups."""
    groups = [(0, 700, 1), (700, 129, 2), (900, 1, 7), (100, 1025, 0), (1000, 600, 40), (5, 64, 3)]
    n = 2 + sum(c for _, _, c in groups) + 3
    lens = [0, 1, 2, 63, 64, 65, 130, 511, 512, 513, 17, 300]
    own = [((37 * i) % 900, lens[i % len(lens)]) for i in range(n)]
    c = Case(gpu, dtype, H, Hkv, Dh, 1700, groups, own, lead=2, seed=H + Dh)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("P", [0, 1, 31, 32, 33, 127, 128, 129, 255, 257, 1023, 1024, 1025, 2049, 5000])
def test_prefix_lengths(gpu, dtype, P):
    own = [(5000, L) for L in (0, 1, 31, 33, 512, 700)]
    c = Case(gpu, dtype, 4, 2, 64, 5700, [(0, P, 6)], own, seed=P)
    out = c.run()
    c.check(out)
    assert P > 0 or not out[0].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv", [(16, 16), (16, 4)])
def test_long_prefix(gpu, dtype, H, Hkv):
    """Past the largest chunk, large scores."""
    own = [(20000 + 16 * i, 5 * i) for i in range(18)]
    c = Case(gpu, dtype, H, Hkv, 128, 20600, [(3, 19990, 18)], own, seed=1, std=4.0)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_blocks_are_the_same_bits(gpu, dtype):
    groups = [(1024, 1000, 5), (0, 333, 4)]
    own = [(2048 + 64 * i, 7 * i) for i in range(9)]
    a = Case(gpu, dtype, 4, 2, 128, 4096, groups, own)
    b = Case(gpu, dtype, 4, 2, 128, 4096, groups, own, block=1024)
    out = a.run()
    a.check(out)
    assert torch.equal(out, b.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv", [(4, 4), (8, 2)])
def test_a_row_does_not_see_its_companions(gpu, dtype, H, Hkv):
    groups = [(0, 1500, 70), (1500, 300, 20)]
    own = [(1800 + i, (11 * i) % 600) for i in range(95)]
    c = Case(gpu, dtype, H, Hkv, 64, 2600, groups, own, seed=3)
    out = c.run()
    assert torch.equal(c.run(), out)
    assert torch.equal(c.run(prefix_len_max=2500, kv_len_max=2600, group_max=None), out)
    for rows in ([0], [69], [70], [94], [3, 17, 40, 71, 90], list(range(33)), list(range(20, 95))):
        assert torch.equal(c.run(rows), out[rows])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_groups_and_no_keys(gpu, dtype):
    c = Case(gpu, dtype, 4, 2, 64, 600, [], [(0, 20), (10, 0), (20, 512), (3, -4)])
    out = c.run()
    c.check(out)
    assert not out[1].any() and not out[3].any()
    c = Case(gpu, dtype, 4, 2, 64, 100, [(0, 0, 2), (4, -1, 1)], [(0, 0)] * 3)
    assert not c.run().any()
    assert not c.run(prefix_len_max=50, kv_len_max=50).any()
    z = lambda d: torch.empty(0, dtype=d, device=gpu)  # noqa: E731
    a = c.args()
    empty = ops.attn_shared(a[0][:0], *a[1:3], z(torch.int64), z(torch.int32), torch.zeros(1, dtype=torch.int32,
                            device=gpu), z(torch.int64), z(torch.int32), prefix_len_max=0, kv_len_max=0)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_special_values_stay_with_the_rows_that_attend_them(gpu, dtype, bad):
    groups = [(0, 300, 20), (400, 150, 20)]
    own = [(600 + 3 * i, 1 + i) for i in range(40)]
    c = Case(gpu, dtype, 4, 2, 64, 800, groups, own, seed=4)
    want = c.run()
    for t in (c.k, c.v):  # next to the prefixes' and the rows' last keys, and between them
        t[300:400], t[550:600], t[758:] = bad, bad, bad
    assert torch.equal(c.run(), want)
    c.v[299, 0, 5] = bad   # last key of the first prefix, kv head 0
    c.k[602, 1] = math.nan  # own key 2 of row 0 (not attended: one key), own key of no other row's start
    got = c.run()
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[:20, :2, 5] = True
    assert bool((~torch.isfinite(got[hit])).all())
    for i in range(40):
        if 602 in c.keys(i):
            hit[i, 2:] = True
            assert bool(got[i, 2:].isnan().all())
    assert torch.equal(got[~hit], want[~hit])


def test_rows_past_32_bit_offsets(gpu):
    Dh, rows = 128, (1 << 25) + 2048  # more than 2^32 elements
    k, v = (torch.empty(rows, 1, Dh, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    g = _gen(5)
    tail = [torch.randn(2048, 1, Dh, generator=g).bfloat16() for _ in range(2)]
    for t, x in zip((k, v), tail):
        t[-2048:] = x.to(gpu)
    q = torch.randn(3, 2, Dh, generator=g).bfloat16()
    d = lambda x, dt: torch.tensor(x, dtype=dt, device=gpu)  # noqa: E731
    base = rows - 2048
    out = ops.attn_shared(q.to(gpu), k, v, d([base], torch.int64), d([1500], torch.int32), d([0, 3], torch.int32),
                          d([base + 1500 + 100 * i for i in range(3)], torch.int64), d([90, 0, 5], torch.int32),
                          prefix_len_max=1500, kv_len_max=90)
    for i, L in enumerate((90, 0, 5)):
        at = list(range(1500)) + list(range(1500 + 100 * i, 1500 + 100 * i + L))
        check_attention(out[i], *attend(q[i].double(), tail[0][at].double().transpose(0, 1),
                                        tail[1][at].double().transpose(0, 1), 1 / math.sqrt(Dh), 2.0 ** -8))


@pytest.mark.parametrize("scale", [0.5, 0.0, -0.2])
def test_scale_out_and_workspace(gpu, scale):
    c = Case(gpu, torch.bfloat16, 4, 4, 64, 900, [(0, 600, 4)], [(600, 50)] * 4, seed=6)
    out = torch.empty_like(c.q, device=gpu)
    ws = torch.empty(ops.attn_shared_workspace_bytes(4, 4, 4, 64, 600, 50), dtype=torch.uint8, device=gpu)
    assert c.run(scale=scale, out=out, workspace=ws) is out
    c.check(out, scale)


def test_captured_call_with_moving_lengths(gpu):
    """One graph over growing answers, beside eager calls on another stream."""
    S = 700
    c = Case(gpu, torch.bfloat16, 8, 2, 128, 1200 + 12 * S, [(0, 1200, 12)], [(1200 + S * i, 1) for i in range(12)])
    a = c.args()
    mx = dict(prefix_len_max=1200, kv_len_max=S, group_max=12)
    ops.attn_shared(*a, **mx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.attn_shared(*a, **mx)
    side = torch.cuda.Stream()
    for step in range(4):
        lens = [1 + (step * 200 + 13 * i) % S for i in range(12)]
        c.own = [(b, L) for (b, _), L in zip(c.own, lens)]
        a[7].copy_(torch.tensor(lens, dtype=torch.int32))
        a[4].copy_(torch.tensor([1200 - 17 * step], dtype=torch.int32))
        c.groups = [(0, 1200 - 17 * step, 12)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = ops.attn_shared(*a, **mx)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)
        c.check(eager)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv,Dh", [(4, 4, 64), (8, 2, 128)])
def test_infinities_in_v_come_out_as_themselves(gpu, dtype, H, Hkv, Dh):
    """An infinity in V is the row's result in that column, opposite ones and NaN are NaN, and
    every other value keeps its bits, beside a row whose query is NaN too."""
    groups = [(0, 900, 30), (900, 40, 12)]
    own = [(1000 + 5 * i, (7 * i) % 60) for i in range(42)]
    c = Case(gpu, dtype, H, Hkv, Dh, 1300, groups, own, seed=Dh)
    c.q[4, H - 1, 3] = math.nan
    want = c.run().cpu()
    c.v[17, 0, 1] = c.v[899, 0, 1] = c.v[300, 0, 2] = math.inf
    c.v[18, 0, 3] = c.v[400, 0, 4] = c.v[899, 0, 4] = -math.inf
    c.v[300, 0, 5], c.v[301, 0, 5], c.v[310, 0, 6] = math.inf, -math.inf, math.nan
    c.v[500, 0, 7], c.v[501, 0, 7] = math.inf, math.nan
    c.v[905, Hkv - 1, :8] = math.inf
    c.v[1000 + 5 * 9, 0, 8] = -math.inf  # a row's own key
    got = c.run().cpu()
    infinite = 0
    for i in range(42):
        at = c.keys(i)
        ref, _ = attend(c.q[i].double(), c.k[at].double().transpose(0, 1), c.v[at].double().transpose(0, 1),
                        1 / math.sqrt(Dh))
        special = ~torch.isfinite(ref)
        infinite += int(ref.isinf().sum())
        assert torch.equal(got[i][special].double().nan_to_num(nan=7.0), ref[special].nan_to_num(nan=7.0))
        assert torch.equal(got[i][~special], want[i][~special])
    assert infinite > 200


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_workgroups_than_a_grid_row(gpu, dtype):
    """Empty groups, and bounds far above the lengths, until the workgroups pass 2^24: the
    bits of the call that counts only what is there."""
    groups = [(0, 1100, 300), (1100, 77, 200)]
    own = [(1200 + i, i % 40) for i in range(512)]
    c = Case(gpu, dtype, 16, 4, 64, 1800, groups, own, seed=7)
    want = c.run()
    q, k, v, base, length, first, *rest = c.args()
    empty = 2098  # groups between the two
    base, length = (torch.cat([t[:1], t[1:].expand(empty), t[1:]]) for t in (base, length))
    first = torch.cat([first[:1], first[1:2].expand(empty + 1), first[2:]])
    got = ops.attn_shared(q, k, v, base, length, first, *rest, prefix_len_max=32768, kv_len_max=600)
    assert torch.equal(got, want)


def test_bounds_of_the_largest_length(gpu):
    """2^31 - 1 as "no bound": every key counts, the bits are those of close bounds."""
    c = Case(gpu, torch.bfloat16, 1, 1, 64, 42000, [(0, 40000, 2)], [(40000, 1500), (41000, 7)], seed=8)
    want = c.run()
    top = 2 ** 31 - 1
    ws = torch.empty(ops.attn_shared_workspace_bytes(2, 1, 1, 64, top, top), dtype=torch.uint8, device=gpu)  # 3.3 GB
    assert torch.equal(c.run(prefix_len_max=top, kv_len_max=top, workspace=ws), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group_max", [0, 1, 7, 8, 9, 30])
def test_rows_past_group_max_are_nan(gpu, dtype, group_max):
    """Nothing was computed for them: not a merge of what the workspace held. Rows of an
    empty prefix, and rows of no group, need no prefix and are what they are."""
    groups = [(0, 500, 40), (500, 200, 8), (700, 0, 35)]
    own = [(800 + i, 1 + i % 20) for i in range(90)]
    c = Case(gpu, dtype, 8, 2, 64, 1000, groups, own, seed=9)
    want = c.run()
    ws = torch.zeros(ops.attn_shared_workspace_bytes(90, 8, 2, 64, 500, 20), dtype=torch.uint8, device=gpu)
    got = c.run(group_max=group_max, workspace=ws)
    lost = torch.zeros(90, dtype=torch.bool)
    lost[group_max:40] = True
    lost[40 + group_max:48] = True
    assert bool(got[lost].isnan().all()) and torch.equal(got[~lost], want[~lost])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_nan_scale_gives_nan(gpu, dtype):
    c = Case(gpu, dtype, 8, 2, 128, 900, [(0, 600, 5), (600, 0, 2)], [(600 + 9 * i, 8 * (i % 3)) for i in range(9)])
    got = c.run(scale=math.nan)
    keys = torch.tensor([len(c.keys(i)) > 0 for i in range(9)])
    assert not bool(keys.all()) and bool(got[keys].isnan().all()) and not bool(got[~keys].any())


def test_rows_past_32_bit_offsets_to_the_last_bits(gpu):
    """The bound of two bf16 terms a probability, far into a cache, in both layouts."""
    Dh, rows, B = 64, (1 << 26) + 4096, 2048  # more than 2^32 elements
    g = _gen(11)
    tail = [torch.randn(B, 1, Dh, generator=g).bfloat16() for _ in range(2)]
    q = torch.randn(3, 2, Dh, generator=g).bfloat16()
    d = lambda x, dt: torch.tensor(x, dtype=dt, device=gpu)  # noqa: E731
    base, outs = rows - B, []
    for shape in ((rows, 1, Dh), (rows // B, 1, B, Dh)):
        k, v = (torch.empty(shape, dtype=torch.bfloat16, device=gpu) for _ in range(2))
        for t, x in zip((k, v), tail):
            t.view(rows, 1, Dh)[-B:] = x.to(gpu)
        outs.append(ops.attn_shared(q.to(gpu), k, v, d([base], torch.int64), d([1500], torch.int32),
                                    d([0, 3], torch.int32), d([base + 1500 + 100 * i for i in range(3)], torch.int64),
                                    d([90, 0, 5], torch.int32), prefix_len_max=1500, kv_len_max=90))
        del k, v
    assert torch.equal(*outs)
    for i, L in enumerate((90, 0, 5)):
        at = list(range(1500)) + list(range(1500 + 100 * i, 1500 + 100 * i + L))
        check_attention(outs[0][i], *attend(q[i].double(), tail[0][at].double().transpose(0, 1),
                                            tail[1][at].double().transpose(0, 1), 1 / math.sqrt(Dh),
                                            P_STEP[torch.bfloat16]))
