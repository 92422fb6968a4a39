"""The 8-bit slot cache and its decode attention on the GPU, against their definitions in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from tests.serving_ref import CODE_DTYPES, attend, check_attention, quantise, rotate
from wavefront_decoding_amd import ops

pytestmark = pytest.mark.gpu

CODES = ["e4m3", "int8"]
DTYPES = [torch.bfloat16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache(rows, Hkv, Dh, code, gpu, block=0):
    """block: rows per head-major block (0: token-major)."""
    shape = (rows, Hkv, Dh) if not block else (rows // block, Hkv, block, Dh)
    return ops.QuantKV.zeros(shape, code=CODE_DTYPES[code], device=gpu)


def _hard_rows(n, Hkv, Dh, code, dtype, seed):
    """Rows of every magnitude; values on the borders between codes; largest values on
    and next to the exponent's border; zeros, denormals."""
    g = _gen(seed)
    x = torch.randn(n, Hkv, Dh, generator=g, dtype=torch.float64)
    x *= torch.exp2(torch.randint(-100, 100, (n, Hkv, 1), generator=g).double())
    for i in range(0, n, 3):  # a small grid: many ties
        x[i] = torch.randint(-64, 65, (Hkv, Dh), generator=g).double() * 2.0 ** (i % 7 - 3) / 8
    c = 448.0 if code == "e4m3" else 127.0
    if n > 8:
        x[4] = x[4].clamp(-1, 1)
        x[4, :, 0] = c * 2.0 ** -5                  # exactly on the border
        x[5] = x[4]
        x[5, :, 0] = c * 2.0 ** -5 * (1 + 2.0 ** (-7 if dtype == torch.bfloat16 else -23))  # one step above
        x[6] = 0.0
        x[7] = torch.randn(Hkv, Dh, generator=g).double() * 2.0 ** -128  # denormals
        x[8] = torch.randn(Hkv, Dh, generator=g).double() * 2.0 ** -140
    return x.to(dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,Hkv,Dh,block", [(1, 1, 64, 0), (7, 3, 128, 0), (9, 16, 128, 64), (131, 4, 64, 32),
                                            (300, 2, 128, 512)])
def test_append_then_read(gpu, code, dtype, n, Hkv, Dh, block):
    rows = 1024
    cache = _cache(rows, Hkv, Dh, code, gpu, block)
    k, v = (_hard_rows(n, Hkv, Dh, code, dtype, s) for s in (n, n + 1))
    at = torch.randperm(rows, generator=_gen(n))[:n]
    ops.kv_append_q(k.to(gpu), v.to(gpu), cache, at.to(gpu))
    for out_dtype in DTYPES:
        gk, gv = ops.kv_read_q(cache, at.to(gpu), dtype=out_dtype)
        for got, x in ((gk, k), (gv, v)):
            assert torch.equal(got.cpu(), quantise(x, code)[0].to(out_dtype))
    # the exponents are the definition's, and no other row was touched
    exps = cache.k_exp.cpu()
    exps = exps.reshape(rows, Hkv) if not block else exps.permute(0, 2, 1).reshape(rows, Hkv)
    assert torch.equal(exps[at].int() - 127, quantise(k, code)[1].int())
    rest = torch.ones(rows, dtype=torch.bool)
    rest[at] = False
    other = rest.nonzero().flatten().to(gpu)
    for t in ops.kv_read_q(cache, other, dtype=torch.float32):
        assert not t.any()
    assert (exps[rest] == 1).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_with_infinities_or_nan_read_as_nan_alone(gpu, code, dtype):
    n, Hkv, Dh = 6, 2, 64
    k = torch.randn(n, Hkv, Dh, generator=_gen(3)).to(dtype)
    v = torch.randn(n, Hkv, Dh, generator=_gen(4)).to(dtype)
    k[1, 0, 5], k[2, 1, 63], v[3, 0, 0] = math.inf, math.nan, -math.inf
    cache = _cache(n, Hkv, Dh, code, gpu)
    rows = torch.arange(n, device=gpu)
    ops.kv_append_q(k.to(gpu), v.to(gpu), cache, rows)
    gk, gv = (t.cpu() for t in ops.kv_read_q(cache, rows, dtype=dtype))
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got.isnan().all(-1), ~torch.isfinite(x).all(-1))
        assert torch.equal(got.isnan().any(-1), ~torch.isfinite(x).all(-1))
        assert torch.allclose(got, quantise(x, code)[0].to(dtype), rtol=0, atol=0, equal_nan=True)


def test_append_views_of_a_fused_row(gpu):
    n, H, Hkv, Dh = 37, 4, 2, 64
    qkv = torch.randn(n, (H + 2 * Hkv) * Dh, generator=_gen(5)).bfloat16().to(gpu)
    x = qkv.view(n, H + 2 * Hkv, Dh)
    k, v = x[:, H: H + Hkv], x[:, H + Hkv:]
    a, b = (_cache(64, Hkv, Dh, "e4m3", gpu) for _ in range(2))
    rows = torch.randperm(64, generator=_gen(6))[:n].to(gpu)
    ops.kv_append_q(k, v, a, rows)
    ops.kv_append_q(k.contiguous(), v.contiguous(), b, rows)
    for s, t in zip(a.tensors, b.tensors):
        assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,Hkv,Dh,block", [(1, 4, 4, 64, 0), (33, 4, 2, 64, 16), (130, 16, 4, 128, 0),
                                              (19, 3, 1, 128, 32)])
def test_rope_append(gpu, code, dtype, n, H, Hkv, Dh, block):
    g = _gen(n + H)
    pitch = (H + 2 * Hkv) * Dh + 32
    qkv = (torch.randn(n, pitch, generator=g) * torch.exp2(torch.randint(-6, 6, (n, 1), generator=g))).to(dtype)
    S = 5000
    ang = torch.arange(S).double()[:, None] * 10000.0 ** (-2.0 * torch.arange(Dh // 2).double() / Dh)[None]
    cos, sin = ang.cos().float(), ang.sin().float()
    pos = torch.randint(0, S, (n,), generator=g)
    rows = torch.randperm(160, generator=g)[:n]
    cache = _cache(160, Hkv, Dh, code, gpu, block)
    x = qkv.to(gpu)[:, : (H + 2 * Hkv) * Dh]
    args = (x, pos.int().to(gpu), cos.to(gpu), sin.to(gpu), rows.to(gpu))
    q = ops.qkv_rope_append_q(*args, cache, H, Hkv, Dh)
    # q: the bits of the unquantised path
    kc = torch.zeros((160, Hkv, Dh) if not block else (160 // block, Hkv, block, Dh), dtype=dtype, device=gpu)
    assert torch.equal(q, ops.qkv_rope_append(*args, kc, kc.clone(), H, Hkv, Dh))
    heads = qkv[:, : (H + 2 * Hkv) * Dh].view(n, H + 2 * Hkv, Dh)
    k = rotate(heads[:, H: H + Hkv], cos[pos], sin[pos])
    gk, gv = ops.kv_read_q(cache, rows.to(gpu), dtype=torch.float32)
    assert torch.equal(gk.cpu().double(), quantise(k, code)[0])
    assert torch.equal(gv.cpu().double(), quantise(heads[:, H + Hkv:], code)[0])


def test_rows_past_32_bit_offsets(gpu):
    """Codes beyond 4 GiB, exponents with them; both layouts."""
    Dh, rows = 128, (1 << 25) + 64
    for shape in ((rows, 1, Dh), (rows // 64, 1, 64, Dh)):
        codes = [torch.empty(shape, dtype=torch.int8, device=gpu) for _ in range(2)]
        exps = [torch.empty(shape[:-1], dtype=torch.uint8, device=gpu) for _ in range(2)]
        cache = ops.QuantKV(*codes, *exps)
        at = torch.cat([torch.arange(rows - 50, rows), torch.arange(7)])
        k, v = (torch.randn(57, 1, Dh, generator=_gen(s)).bfloat16() for s in (1, 2))
        ops.kv_append_q(k.to(gpu), v.to(gpu), cache, at.to(gpu))
        gk, gv = ops.kv_read_q(cache, at.to(gpu), dtype=torch.float32)
        for got, x in ((gk, k), (gv, v)):
            assert torch.equal(got.cpu().double(), quantise(x, "int8")[0])
        q = torch.randn(1, 1, Dh, generator=_gen(3)).bfloat16()
        base, n = rows - 50, 50
        out = ops.attn_decode_q(q.to(gpu), cache, torch.tensor([base], device=gpu),
                                torch.tensor([n], dtype=torch.int32, device=gpu), kv_len_max=64)
        ref, bound = attend(q[0].double(), gk[:50, 0].cpu().double()[None], gv[:50, 0].cpu().double()[None],
                            1 / math.sqrt(Dh))
        check_attention(out[0], ref, bound)
        del cache, codes, exps


def _filled(rows, Hkv, Dh, code, gpu, seed, block=0):
    cache = _cache(rows, Hkv, Dh, code, gpu, block)
    g = _gen(seed)
    k, v = (torch.randn(rows, Hkv, Dh, generator=g).bfloat16() for _ in range(2))
    at = torch.arange(rows, device=gpu)
    ops.kv_append_q(k.to(gpu), v.to(gpu), cache, at)
    return cache, [t.double().cpu() for t in ops.kv_read_q(cache, at, dtype=torch.float32)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,Dh,block", [(4, 4, 64, 0), (4, 2, 64, 2600), (8, 2, 128, 0), (3, 3, 128, 2600),
                                            (4, 2, 128, 2600), (4, 1, 64, 0), (16, 1, 128, 0), (10, 2, 64, 2600)])
def test_attention_lengths_and_layouts(gpu, code, dtype, H, Hkv, Dh, block):
    """Lengths around a tile, a split and the zero row; each row as if it were alone."""
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 500, 1023, 1024, 1025, 2049, 2600, -3]
    slots = 3
    cache, (k, v) = _filled(slots * 2600, Hkv, Dh, code, gpu, Dh + H, block)
    n = len(lens)
    q = (torch.randn(n, H, Dh, generator=_gen(9)) * 2).to(dtype)
    base = torch.tensor([2600 * (i % slots) for i in range(n)])
    args = lambda i: (base[i].to(gpu), torch.tensor(lens, dtype=torch.int32)[i].to(gpu))  # noqa: E731
    out = ops.attn_decode_q(q.to(gpu), cache, *args(slice(None)), kv_len_max=2600)
    for i, L in enumerate(lens):
        span = slice(int(base[i]), int(base[i]) + max(L, 0))
        ref, bound = attend(q[i].double(), k[span].transpose(0, 1), v[span].transpose(0, 1), 1 / math.sqrt(Dh),
                            2.0 ** -16 if dtype == torch.bfloat16 else 0.0)
        check_attention(out[i], ref, bound)
        one = slice(i, i + 1)
        alone = ops.attn_decode_q(q[one].to(gpu), cache, *args(one), kv_len_max=2600)
        assert torch.equal(alone[0], out[i])
    assert not out[0].any() and not out[-1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,Dh", [(8, 4, 64), (16, 4, 128)])
def test_attention_of_many_rows_is_that_of_each_alone(gpu, dtype, H, Hkv, Dh):
    """Rows enough that a workgroup takes all splits of one: the bits of a row alone, whose
    splits are merged by another launch, and of a call whose longest row could be longer."""
    S, n = 4000, 150
    cache, (k, v) = _filled(2 * S, Hkv, Dh, "int8", gpu, 3)
    g = _gen(Dh)
    lens = torch.randint(-1, S + 1, (n,), generator=g)
    lens[:8] = torch.tensor([0, 1, 1024, 1025, 2048, 2049, S, -5])
    base = torch.randint(0, S, (n,), generator=g)
    q = (torch.randn(n, H, Dh, generator=g) * 2).to(dtype)
    args = lambda at: (q[at].to(gpu), cache, base[at].to(gpu), lens[at].int().to(gpu))  # noqa: E731
    out = ops.attn_decode_q(*args(slice(None)), kv_len_max=S)
    assert torch.equal(ops.attn_decode_q(*args(slice(None)), kv_len_max=2 * S), out)
    for i in [*range(12), 60, 149]:
        assert torch.equal(ops.attn_decode_q(*args(slice(i, i + 1)), kv_len_max=S)[0], out[i])
        span = slice(int(base[i]), int(base[i]) + max(int(lens[i]), 0))
        check_attention(out[i], *attend(q[i].double(), k[span].transpose(0, 1), v[span].transpose(0, 1),
                                        1 / math.sqrt(Dh), 2.0 ** -16 if dtype == torch.bfloat16 else 0.0))


@pytest.mark.parametrize("code", CODES)
def test_attention_reads_no_row_past_its_length(gpu, code):
    """Rows behind the length hold NaN codes and the non-finite mark: no effect. A
    marked row within it makes the rows that attend it NaN, no others."""
    H, Hkv, Dh, S = 4, 2, 64, 200
    cache, _ = _filled(S, Hkv, Dh, code, gpu, 1)
    lens = torch.tensor([70, 100, 130], dtype=torch.int32, device=gpu)
    base = torch.zeros(3, dtype=torch.int64, device=gpu)
    q = torch.randn(3, H, Dh, generator=_gen(2)).bfloat16().to(gpu)
    want = ops.attn_decode_q(q, cache, base, lens, kv_len_max=S)
    for t, x in zip(cache.tensors, (0x7f, 0x7f, 255, 255)):
        t.view(torch.uint8)[130:] = x
    assert torch.equal(ops.attn_decode_q(q, cache, base, lens, kv_len_max=S), want)
    cache.k_exp[100, 0] = 255  # row 100 of kv head 0: query heads 0, 1 of the last row only
    got = ops.attn_decode_q(q, cache, base, lens, kv_len_max=S)
    assert bool(torch.equal(got[:2], want[:2]) and torch.equal(got[2, 2:], want[2, 2:]))
    assert bool(got[2, :2].isnan().all())


def test_attention_marked_row_reaches_rows_of_several_splits(gpu):
    H, Hkv, Dh, S = 2, 2, 128, 3000
    cache, _ = _filled(S, Hkv, Dh, "e4m3", gpu, 1)
    cache.v_exp[2500, 1] = 255
    lens = torch.tensor([3000, 2500], dtype=torch.int32, device=gpu)
    q = torch.randn(2, H, Dh, generator=_gen(2)).bfloat16().to(gpu)
    nan = ops.attn_decode_q(q, cache, torch.zeros(2, dtype=torch.int64, device=gpu), lens, kv_len_max=S).isnan()
    assert bool(nan[0, 1].all()) and not bool(nan[0, 0].any()) and not bool(nan[1].any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attention_any_scale_and_large_scores(gpu, dtype, scale):
    H, Hkv, Dh, S = 4, 2, 64, 1100
    cache, (k, v) = _filled(S, Hkv, Dh, "int8", gpu, 5)
    q = (torch.randn(3, H, Dh, generator=_gen(4)) * 3).to(dtype)
    lens = [1100, 40, 7]
    got = ops.attn_decode_q(q.to(gpu), cache, torch.zeros(3, dtype=torch.int64, device=gpu),
                            torch.tensor(lens, dtype=torch.int32, device=gpu), kv_len_max=S, scale=scale)
    for i, L in enumerate(lens):
        check_attention(got[i], *attend(q[i].double(), k[:L].transpose(0, 1), v[:L].transpose(0, 1), scale,
                                        2.0 ** -16 if dtype == torch.bfloat16 else 0.0))


def test_attention_scale_and_workspace_and_out(gpu):
    H, Hkv, Dh, S = 4, 4, 128, 1500
    cache, (k, v) = _filled(S, Hkv, Dh, "e4m3", gpu, 7)
    q = torch.randn(2, H, Dh, generator=_gen(2)).bfloat16()
    out = torch.empty(2, H, Dh, dtype=torch.bfloat16, device=gpu)
    ws = torch.empty(ops.attn_workspace_bytes(2, H, Dh, S), dtype=torch.uint8, device=gpu)
    got = ops.attn_decode_q(q.to(gpu), cache, torch.zeros(2, dtype=torch.int64, device=gpu),
                            torch.tensor([S, 3], dtype=torch.int32, device=gpu), kv_len_max=S, scale=0.31, out=out,
                            workspace=ws)
    assert got is out
    for i, L in enumerate((S, 3)):
        check_attention(got[i], *attend(q[i].double(), k[:L].transpose(0, 1), v[:L].transpose(0, 1), 0.31))


def test_captured_tick(gpu):
    """Rotate, write and attend inside one graph, replayed with new rows, lengths and
    positions, beside eager calls on another stream."""
    n, H, Hkv, Dh, S = 5, 4, 2, 64, 1200
    cache, _ = _filled(n * S, Hkv, Dh, "e4m3", gpu, 3, block=S)
    g = _gen(8)
    cos, sin = (torch.randn(S, Dh // 2, generator=g).to(gpu) for _ in range(2))
    qkv = torch.empty(n, (H + 2 * Hkv) * Dh, dtype=torch.bfloat16, device=gpu)
    pos = torch.empty(n, dtype=torch.int32, device=gpu)
    row, lens = torch.empty(n, dtype=torch.int64, device=gpu), torch.empty(n, dtype=torch.int32, device=gpu)
    base = torch.arange(n, dtype=torch.int64, device=gpu) * S

    def fill(step):
        p = torch.tensor([step, 40 + step, 1000 + step, 1030 + step, 1100 + step], dtype=torch.int32)
        pos.copy_(p)
        row.copy_(base + pos)
        lens.copy_(p + 1)
        qkv.copy_(torch.randn(qkv.shape, generator=_gen(step)))

    def tick(c):
        q = ops.qkv_rope_append_q(qkv, pos, cos, sin, row, c, H, Hkv, Dh)
        return ops.attn_decode_q(q, c, base, lens, kv_len_max=S)

    twin = ops.QuantKV(*(t.clone() for t in cache.tensors))
    fill(0)
    tick(twin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = tick(cache)
    side = torch.cuda.Stream()
    for step in range(4):
        fill(step)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = tick(twin)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)
        for a, b in zip(cache.tensors, twin.tensors):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_empty_calls(gpu):
    cache = _cache(8, 2, 64, "e4m3", gpu)
    z = lambda *s, d=torch.bfloat16: torch.empty(*s, dtype=d, device=gpu)  # noqa: E731
    ops.kv_append_q(z(0, 2, 64), z(0, 2, 64), cache, z(0, d=torch.int64))
    assert ops.kv_read_q(cache, z(0, d=torch.int64))[0].shape == (0, 2, 64)
    assert ops.attn_decode_q(z(0, 4, 64), cache, z(0, d=torch.int64), z(0, d=torch.int32), kv_len_max=4).shape[0] == 0
    cos = z(4, 32, d=torch.float32)
    assert ops.qkv_rope_append_q(z(0, 512), z(0, d=torch.int32), cos, cos, z(0, d=torch.int64), cache, 4, 2,
                                 64).shape == (0, 4, 64)


def test_cache_tensors_moved_in_place(gpu):
    """The kernels work where the cache's tensors are, not where they were."""
    n, Hkv, Dh = 9, 2, 64
    cache = _cache(16, Hkv, Dh, "int8", gpu)
    k, v = (torch.randn(n, Hkv, Dh, generator=_gen(s)).bfloat16() for s in (1, 2))
    rows = torch.arange(n, device=gpu)
    ops.kv_append_q(k.to(gpu), v.to(gpu), cache, rows)
    old = cache.k.data
    before = old.clone()
    cache.k.data = torch.zeros_like(old)
    ops.kv_append_q(v.to(gpu), v.to(gpu), cache, rows)
    assert torch.equal(old, before)
    for got in ops.kv_read_q(cache, rows):
        assert torch.equal(got.cpu(), quantise(v, "int8")[0].bfloat16())
