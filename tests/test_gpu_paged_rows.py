"""Rows of the paged attention on the GPU: a draft's rows have the bits of the single tokens that they verify."""
from __future__ import annotations

import pytest
import torch

from tests.paged_ref import Pages
from wavefront_decoding_amd import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]
# (H, Hkv, Dh), and lengths at which drafts of these heads end: at edges of blocks, of parts of 512 and 1024 keys, and
# in sequences of more than sixteen parts
SHAPES = [((16, 16, 128), (5, 33, 511, 520, 768, 769, 1030, 2049, 2070, 3080, 5000)),
          ((16, 4, 128), (40, 513, 770, 1024, 6000, 8195, 9220, 12000)),
          ((4, 4, 64), (64, 513, 700, 1025, 8200, 9000)),
          ((8, 1, 64), (100, 600, 7000, 9000, 20000, 33000)),
          ((10, 2, 64), (30, 515, 16390, 17500))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4), (1000, 0), (1030, 700), (9500, 20)])
@pytest.mark.parametrize("heads,ends", SHAPES)
def test_a_draft_has_the_bits_of_single_tokens(gpu, dtype, window, sinks, heads, ends):
    """Rows verified together and the same rows one at a time, each as the newest of its context."""
    H, Hkv, Dh = heads
    most = 64 // (H // Hkv)
    seqs = [(min(L, m), L) for L in ends for m in (2, 9, most) if m <= most]
    c = Pages(gpu, dtype, H, Hkv, Dh, seqs, page=64, seed=H)
    drafts = c.attn(window=window, sinks=sinks)
    rows = [(b, L - m + i + 1) for b, (m, L) in enumerate(seqs) for i in range(m)]
    n = len(rows)
    table = c.table[torch.tensor([b for b, _ in rows], device=gpu)]
    one = ops.attn_paged(c.q, c.k, c.v, table, torch.arange(n + 1, dtype=torch.int32, device=gpu),
                         c.ints([p for _, p in rows]), q_len_max=1, kv_len_max=c.kv_len_max, window=window,
                         sinks=sinks)
    same = (drafts == one).flatten(1).all(-1).tolist()
    assert all(same), [(seqs[b], p) for (b, p), ok in zip(rows, same) if not ok][:5]


@pytest.mark.parametrize("dtype", DTYPES)
def test_bounds_change_no_bits(gpu, dtype):
    """kv_len_max decides whether a window covers every key, and the workspace: neither shows in a row."""
    c = Pages(gpu, dtype, 32, 32, 64, [(1, 2500), (2, 1400), (1, 40), (1, 2900)], page=64, table_pad=100)
    for window, sinks in ((0, 0), (3000, 0), (2900, 5), (1500, 9)):
        ref = c.attn(window=window, sinks=sinks)
        for most in (2901, 3000, 3001, 9000):
            assert torch.equal(ref, c.attn(window=window, sinks=sinks, kv_len_max=most)), (window, most)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,Dh", [(16, 16, 64), (16, 4, 64), (8, 1, 64), (32, 1, 128), (6, 6, 128)])
def test_parts_stay_in_the_workspace(gpu, dtype, H, Hkv, Dh):
    """Calls of few and many rows with a workspace of just the named size, between bytes that stay as they are: the bits
    of the same calls with one of their own."""
    for seed, seqs in enumerate(([(300, 4000)], [(1, 9000), (3, 700)], [(70, 3000), (1, 1200), (9, 2500), (200, 200)],
                                 [(1, 600 + 40 * i) for i in range(20)] + [(33, 2100)], [(65, 8000)] * 3)):
        c = Pages(gpu, dtype, H, Hkv, Dh, seqs, page=64, seed=seed)
        for window, sinks in ((0, 0), (700, 40)):
            need = ops.attn_paged_workspace_bytes(c.n, len(seqs), H, Hkv, Dh, dtype, c.q_len_max, c.kv_len_max, window,
                                                  sinks)
            ws = torch.full((need + 8192,), 0x5a, dtype=torch.uint8, device=gpu)
            got = c.attn(window=window, sinks=sinks, workspace=ws[4096: 4096 + need])
            assert (ws[:4096] == 0x5a).all() and (ws[4096 + need:] == 0x5a).all(), (seqs[:3], window)
            assert torch.equal(got, c.attn(window=window, sinks=sinks))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_hundreds_of_sequences(gpu, dtype, window, sinks):
    """The search for a row's sequence takes 64 sequences a step: rows of few and of many, empty sequences and ones
    without new rows spread over several steps, parts among them."""
    seqs = [((0, 1, 1, 3, 0, 1)[i % 6], 5 + (37 * i) % 400) for i in range(230)]
    for i, seq in ((3, (90, 400)), (62, (1, 1500)), (63, (70, 90)), (64, (1, 2000)), (128, (100, 1800)), (140, (0, 0)),
                   (191, (20, 700)), (192, (1, 1)), (228, (120, 600)), (229, (2, 3000))):
        seqs[i] = seq
    c = Pages(gpu, dtype, 2, 1, 64, seqs, page=32, seed=2, lead=2, tail=3)
    out = torch.full_like(c.q, 7.0)
    c.attn(out=out, window=window, sinks=sinks)
    c.check(out, window=window, sinks=sinks, p_step=2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    assert (out[:2] == 7.0).all() and (out[c.cu[-1]:] == 7.0).all()
    for b in (62, 63, 64, 127, 128, 191, 192, 229):
        m, L = seqs[b]
        one = ops.attn_paged(c.q[c.cu[b]: c.cu[b + 1]].clone(), c.k, c.v, c.table[b: b + 1], c.ints([0, m]), c.ints([L]),
                             q_len_max=max(m, 1), kv_len_max=L, window=window, sinks=sinks)
        assert torch.equal(one, out[c.cu[b]: c.cu[b + 1]]), b


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4), (1030, 700)])
@pytest.mark.parametrize("heads,seqs", [((16, 16, 128), [(200, 2700), (1, 900), (130, 130), (65, 600)]),
                                        ((8, 1, 64), [(9, 700), (60, 9000), (100, 100)]),
                                        ((32, 1, 64), [(3, 40), (16, 1500), (1, 513)]),
                                        ((4, 2, 128), [(600, 600), (70, 17500), (0, 30)])])
def test_by_row_every_row_has_the_bits_of_a_single_token(gpu, dtype, window, sinks, heads, seqs):
    """Drafts, pieces of prompts and whole prompts, and the same rows one at a time."""
    H, Hkv, Dh = heads
    c = Pages(gpu, dtype, H, Hkv, Dh, seqs, page=64, seed=H, lead=1, tail=2)
    out = torch.full_like(c.q, 7.0)
    need = ops.attn_paged_workspace_bytes(c.n, len(seqs), H, Hkv, Dh, dtype, c.q_len_max, c.kv_len_max, window, sinks,
                                          by_row=True)
    ws = torch.full((need + 8192,), 0x5a, dtype=torch.uint8, device=gpu)
    c.attn(out=out, window=window, sinks=sinks, by_row=True, workspace=ws[4096: 4096 + need])
    assert (ws[:4096] == 0x5a).all() and (ws[4096 + need:] == 0x5a).all()
    assert (out[:1] == 7.0).all() and (out[c.cu[-1]:] == 7.0).all()
    rows = [(b, L - m + i + 1) for b, (m, L) in enumerate(seqs) for i in range(m)]
    n = len(rows)
    table = c.table[torch.tensor([b for b, _ in rows], device=gpu)]
    one = ops.attn_paged(c.q[1: 1 + n].clone(), c.k, c.v, table, torch.arange(n + 1, dtype=torch.int32, device=gpu),
                         c.ints([p for _, p in rows]), q_len_max=1, kv_len_max=c.kv_len_max, window=window,
                         sinks=sinks)
    same = (out[1: 1 + n] == one).flatten(1).all(-1).tolist()
    assert all(same), [(seqs[b], p) for (b, p), ok in zip(rows, same) if not ok][:5]


@pytest.mark.parametrize("dtype", DTYPES)
def test_by_row_edges(gpu, dtype):
    """Rows before position 0, past the bounds and of pages outside the pool, as without it."""
    seqs = [(200, 70), (5, 3), (100, 300), (90, 200), (40, -7), (300, 900)]
    c = Pages(gpu, dtype, 4, 2, 64, seqs, page=16, seed=8)
    c.check(c.attn(by_row=True), p_step=2.0 ** -15 if dtype == torch.bfloat16 else 0.0)
    plain, mine = (c.attn(q_len_max=95, kv_len_max=250, by_row=x) for x in (False, True))
    assert torch.equal(plain.isnan(), mine.isnan()) and torch.equal(plain == 0, mine == 0)
    c.table[3, 9] = -1
    mine = c.attn(by_row=True)
    assert torch.equal(mine.isnan(), c.attn().isnan()) and mine[c.cu[3] + 40:c.cu[4]].isnan().all()
