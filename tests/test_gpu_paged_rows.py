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
