"""The serving operators as they are used together: an 8-bit cache's slots, and several
answers to one prompt decoded token by token, eagerly and from one captured graph."""
from __future__ import annotations

import math

import pytest
import torch

from tests.serving_ref import CODE_DTYPES, attend, check_attention, quantise, rotate
from tests.test_gpu_sample import ref_one
from wavefront_decoding_amd import ops
from wavefront_decoding_amd.kv_cache import BatchStaticKVCache, QuantBatchKVCache

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=_gen(seed)).to(dtype)


@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("code", list(CODE_DTYPES))
def test_quant_cache_slots(gpu, code, head_major):
    """Prefill, scattered tokens, read-back, rollback; the trash row is no slot's."""
    cache = QuantBatchKVCache(2, 3, 2, 64, 40, BF16, gpu, head_major=head_major, code=CODE_DTYPES[code])
    assert cache.nbytes == 2 * 2 * 3 * 40 * 2 * 65
    k, v = (_randn(2, 17, 2, 64, seed=s) for s in (1, 2))
    cache.write_prefill(1, k.to(gpu), v.to(gpu), seq_ids=[0, 2])
    tk, tv = (_randn(3, 2, 64, seed=s) for s in (3, 4))
    cache.write_tokens([1, 1, 0], [0, 2, 1], [17, 17, 0], tk.to(gpu), tv.to(gpu))
    junk = torch.full((1, 2, 64), 9.0, dtype=BF16, device=gpu)
    ops.kv_append_q(junk, junk, cache.flat, torch.tensor([cache.trash_row], device=gpu))
    assert [row for row in cache.seqlen] == [[0, 1, 0], [18, 0, 18]]

    def packed(at, want_k, want_v):
        gk, gv, cu, longest = cache.gather_pack(*at)
        lengths = [u + 1 for u in at[2]]
        assert longest == max(lengths) and cu.tolist() == [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        for got, want in ((gk, want_k), (gv, want_v)):
            assert torch.equal(got.cpu(), quantise(torch.cat(want), code)[0].to(BF16))

    at = ([1, 0, 1], [2, 1, 0], [17, 0, 5])
    packed(at, [k[1], tk[1:2], tk[2:3], k[0, :6]], [v[1], tv[1:2], tv[2:3], v[0, :6]])
    cache.drop_positions_at_and_after(2, 10)
    assert cache.seqlen[1] == [18, 0, 10]
    cache.write_tokens([1], [2], [10], tk[:1].to(gpu), tv[:1].to(gpu))
    packed(([1], [2], [10]), [k[1, :10], tk[:1]], [v[1, :10], tv[:1]])
    assert (cache.gather_pack([0], [0], [3])[0] == 0).all()  # never written
    with pytest.raises(IndexError, match="exceeds"):
        cache.write_tokens([0], [0], [40], tk[:1].to(gpu), tv[:1].to(gpu))
    with pytest.raises(IndexError, match="exceeds"):
        cache.write_prefill(0, k[:, :1].expand(2, 41, 2, 64).to(gpu), v[:, :1].expand(2, 41, 2, 64).to(gpu))


class Answers:
    """n answers to one prompt of P tokens, one layer of attention wide: embed, qkv, rotate
    and write, attend, logits, draw. 8-bit: every answer's slot holds the prompt; shared: one
    slot holds it for all."""

    V, D, H, HKV, DH, S = 1008, 256, 4, 2, 64, 400

    def __init__(self, gpu, n, P, code, steps):
        self.n, self.P, self.code = n, P, code
        H, HKV, DH, S, V, D = self.H, self.HKV, self.DH, self.S, self.V, self.D
        dev = lambda t: t.to(gpu)  # noqa: E731
        self.table = dev(_randn(V, D, seed=10))
        self.wqkv = ops.pack_linear(dev(_randn((H + 2 * HKV) * DH, D, seed=11) / 16))
        self.wout = ops.pack_linear(dev(_randn(V, H * DH, seed=12) / 4))
        ang = torch.arange(S).double()[:, None] * 10000.0 ** (-2.0 * torch.arange(DH // 2).double() / DH)[None]
        self.cos, self.sin = dev(ang.cos().float()), dev(ang.sin().float())
        self.u = dev(torch.rand(steps, n, generator=_gen(13)))
        self.temperature = dev(torch.tensor([0.0, 0.7, 1.0, 1.3, 2.0])[torch.arange(n) % 5])
        self.top_k = dev(torch.tensor([0, 40, 0, 1, 300, 7, 1008], dtype=torch.int32)[torch.arange(n) % 7])
        self.top_p = dev(torch.tensor([1.0, 0.9, 0.5])[torch.arange(n) % 3])
        self.ids = dev(-1 - torch.arange(n))
        self.ring_rows = dev(torch.arange(n, dtype=torch.int32))
        self.k, self.v = (_randn(1, P, HKV, DH, seed=s) for s in (14, 15))
        if code:
            self.cache = QuantBatchKVCache(1, n, HKV, DH, S, BF16, gpu, code=CODE_DTYPES[code])
            self.cache.write_prefill(0, dev(self.k.expand(n, -1, -1, -1)), dev(self.v.expand(n, -1, -1, -1)))
        else:
            self.cache = BatchStaticKVCache(1, n + 1, HKV, DH, S, BF16, gpu)
            self.cache.write_prefill(0, dev(self.k), dev(self.v), seq_ids=[n])
            self.prefix = (dev(torch.tensor([self.cache.row_base(0, n)])), dev(torch.tensor([P], dtype=torch.int32)),
                           dev(torch.tensor([0, n], dtype=torch.int32)))
        self.own = P if code else 0  # keys of a slot before the first step
        self.base = dev(torch.tensor([self.cache.row_base(0, b) for b in range(n)]))
        self.pos = torch.empty(n, dtype=torch.int32, device=gpu)
        self.row, self.ring = (torch.empty(n, dtype=torch.int64, device=gpu) for _ in range(2))
        self.lens = torch.empty(n, dtype=torch.int32, device=gpu)
        self.step = torch.empty(1, dtype=torch.int64, device=gpu)
        self.rewind()

    def rewind(self):
        self.pos.fill_(self.P)
        self.row.copy_(self.base + self.own)
        self.lens.fill_(self.own + 1)
        self.ring.copy_(self.ring_rows % self.V)
        self.step.zero_()

    def tick(self):
        n, H, HKV, DH, S = self.n, self.H, self.HKV, self.DH, self.S
        x = ops.embed(self.ids, self.table, ring=self.ring)
        qkv = ops.linear(x, self.wqkv)
        if self.code:
            q = ops.qkv_rope_append_q(qkv, self.pos, self.cos, self.sin, self.row, self.cache.flat, H, HKV, DH)
            o = ops.attn_decode_q(q, self.cache.flat, self.base, self.lens, kv_len_max=S)
        else:
            q = ops.qkv_rope_append(qkv, self.pos, self.cos, self.sin, self.row, self.cache.flat_k,
                                    self.cache.flat_v, H, HKV, DH)
            o = ops.attn_shared(q, self.cache.flat_k, self.cache.flat_v, *self.prefix, self.base, self.lens,
                                prefix_len_max=self.P, kv_len_max=S)
        logits = ops.linear(o.view(n, H * DH), self.wout, out_dtype=torch.float32)
        u = self.u.index_select(0, self.step)[0]
        ids = ops.sample(logits, u, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p,
                         ring=self.ring, ring_rows=self.ring_rows)
        for t in (self.pos, self.row, self.lens, self.step):
            t.add_(1)
        return qkv, q, o, logits, u, ids

    def caches(self):
        return self.cache.flat.tensors if self.code else (self.cache.flat_k, self.cache.flat_v)

    def keys(self, b, length):
        """Row b's keys and values (Hkv, len, Dh) at that length of its slot, 64 bits."""
        if self.code:
            k, v, _, _ = self.cache.gather_pack([0], [b], [length - 1])
        else:
            k, v = (torch.cat([t[0, self.n, :self.P], t[0, b, :length]]) for t in (self.cache.K, self.cache.V))
        return (t.cpu().double().transpose(0, 1) for t in (k, v))

    def check(self, ticks):
        """Every operator of every step, from its own inputs, against its definition."""
        p_step = 2.0 ** -16  # probabilities meet V in two bf16 terms
        H, HKV, DH = self.H, self.HKV, self.DH
        slots = [tuple(self.keys(b, self.own + len(ticks))) for b in range(self.n)]
        for t, (qkv, q, o, logits, u, ids) in enumerate(ticks):
            heads = qkv.cpu().view(self.n, H + 2 * HKV, DH)
            seen = self.P + t + 1
            if self.code:
                k = rotate(heads[:, H: H + HKV], *(x.cpu()[self.P + t].expand(self.n, -1) for x in (self.cos, self.sin)))
                for b in range(self.n):
                    for stored, x in zip(slots[b], (k, heads[:, H + HKV:])):
                        assert torch.equal(stored[:, seen - 1], quantise(x[b], self.code)[0])
            for b in range(self.n):
                ref, bound = attend(q[b].cpu().double(), *(x[:, :seen] for x in slots[b]), 1 / math.sqrt(DH), p_step)
                check_attention(o[b], ref, bound)
            rows, uu = logits.cpu().numpy(), u.tolist()
            par = [x.tolist() for x in (self.temperature, self.top_k, self.top_p)]
            assert ids.tolist() == [ref_one(rows[b], uu[b], par[0][b], par[1][b], par[2][b]) for b in range(self.n)]


@pytest.mark.parametrize("code", ["e4m3", "int8", None], ids=["e4m3", "int8", "shared"])
@pytest.mark.parametrize("n,P", [(1, 1), (5, 63), (35, 300)])
def test_answers_to_one_prompt(gpu, code, n, P):
    steps = 5
    eager, replayed = (Answers(gpu, n, P, code, steps) for _ in range(2))
    eager.tick()  # libraries and workspaces are there before the capture
    eager.rewind()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = replayed.tick()
    replayed.rewind()
    ticks = []
    for _ in range(steps):
        ticks.append([t.clone() for t in eager.tick()])
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, ticks[-1]):
            assert torch.equal(got, want)
        assert torch.equal(eager.ring, replayed.ring) and torch.equal(eager.ring, ticks[-1][-1])
    for a, b in zip(eager.caches(), replayed.caches()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    eager.check(ticks)


def test_answers_are_the_same_alone(gpu):
    """An answer's tokens do not depend on how many are decoded beside it."""
    def tokens(n):
        a = Answers(gpu, 35, 120, "e4m3", 4)
        a.n = n
        for name in ("temperature", "top_k", "top_p", "ids", "ring_rows", "pos", "row", "lens", "base", "ring"):
            setattr(a, name, getattr(a, name)[:n].contiguous())
        a.u = a.u[:, :n].contiguous()
        return torch.stack([a.tick()[-1] for _ in range(4)])

    assert torch.equal(tokens(35)[:, :3], tokens(3))
