"""How many bits of a probability meet V in the paged attention: inputs that show it, what the bounds make of forms with
fewer bits (CPU), and the kernels on them.

Keys come in pairs of nearly the same score whose values are opposite, so an output is the small difference of large
sums: its own rounding hides little, and errors of the probabilities do not cancel."""
from __future__ import annotations

import pytest
import torch

from tests.paged_ref import Pages, attend_rows, check_rows
from tests.serving_ref import HALF_STEP

# bf16 rows of sequences of few rows: P = hi + lo, hi the upper 16 bits of 0.998 P, lo = P - hi rounded. For P in [1, 2)
# lo is below 2^-7 + 0.002 P, so below 2^-6, where a bf16 half step is at most 2^-15.
P_STEP_FEW = {torch.bfloat16: 2.0 ** -15, torch.float32: 0.0}
SEQS = [(1, 24), (1, 200), (4, 64), (8, 700), (3, 1500), (16, 16)]


def paired(dev, dtype, H, Hkv, Dh, seqs, seed=0):
    c = Pages(dev, dtype, H, Hkv, Dh, seqs, page=16, seed=seed)
    g = torch.Generator().manual_seed(seed + 100)
    for b, (_, L) in enumerate(seqs):
        k, v = c.kv[b]
        half = L // 2
        near = k[: 2 * half: 2].float() + 0.02 * torch.randn(half, Hkv, Dh, generator=g)
        k[1: 2 * half: 2] = near.to(dtype)
        v[: 2 * half: 2] = torch.where(torch.rand(half, Hkv, Dh, generator=g) < 0.5, -1.0, 1.0).to(dtype)
        v[1: 2 * half: 2] = -v[: 2 * half: 2]
        for p in range(L):
            at, r = c.place(b, p)
            c.k[at, :, r], c.v[at, :, r] = k[p].to(dev), v[p].to(dev)
    return c


def _cut(x):
    """The upper 16 bits of float32 values."""
    return (x.view(torch.int32) & -65536).view(torch.float32)


FORMS = {
    "two terms": lambda p: _cut(p * 0.998046875) + (p - _cut(p * 0.998046875)).bfloat16().float(),
    "the first term alone": lambda p: _cut(p * 0.998046875),
    "rounded once": lambda p: p.bfloat16().float(),
}


@pytest.mark.parametrize("form", FORMS)
def test_the_bounds_tell_forms_apart(form):
    """Over short contexts; errors of independent roundings average out over many keys."""
    c, worst = paired("cpu", torch.bfloat16, 2, 2, 64, SEQS), []
    for b, (m, L) in enumerate(SEQS):
        q, (k, v) = c.q[c.cu[b]: c.cu[b + 1]], (x.double().transpose(0, 1) for x in c.kv[b])
        pos = torch.arange(L - m, L)
        s = torch.einsum("mhd,hkd->hmk", q.double(), k) * 0.125
        s = s.masked_fill(torch.arange(L) > pos[:, None], -torch.inf)
        # under a reference point that is not the maximum, as the kernels have it
        p = torch.exp(s - s.amax(-1, keepdim=True) + 1.7).float()
        o = (torch.matmul(FORMS[form](p).double(), v) / p.double().sum(-1, keepdim=True)).transpose(0, 1).bfloat16()
        ref, bound = attend_rows(q, *c.kv[b], pos, 0.125, 0, 0, P_STEP_FEW[torch.bfloat16])
        err = (o.double() - ref).abs() / (bound + HALF_STEP[torch.bfloat16] * (ref.abs() + bound))
        worst.append(err.max().item())
    if form == "two terms":
        assert max(worst) <= 1.0, worst
    else:
        assert min(worst[:3]) > 1.5, worst


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv,Dh", [(2, 2, 64), (4, 1, 64), (4, 4, 128), (16, 4, 128)])
def test_probabilities_of_few_rows(gpu, dtype, H, Hkv, Dh):
    c = paired(gpu, dtype, H, Hkv, Dh, SEQS, seed=H)
    for window, sinks in ((0, 0), (300, 4)):
        c.check(c.attn(window=window, sinks=sinks), window=window, sinks=sinks, p_step=P_STEP_FEW[dtype])


@pytest.mark.gpu
def test_probabilities_of_many_rows(gpu):
    """bf16 rows of more than 64 pairs: one rounding to 8 bits; float32 rows of as many: none."""
    seqs = [(70, 300), (200, 200), (130, 1500)]
    for dtype, step in ((torch.bfloat16, 2.0 ** -8), (torch.float32, 0.0)):
        c = paired(gpu, dtype, 4, 4, 64, seqs)
        c.check(c.attn(), p_step=step)
        c.check(c.attn(by_row=True), p_step=P_STEP_FEW[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_random_rows_of_few_rows(gpu, dtype):
    seqs = [(1, 900), (8, 9000), (1, 33), (5, 2000), (16, 600)]
    for std in (1.0, 4.0):
        c = Pages(gpu, dtype, 16, 4, 128, seqs, page=64, seed=11, std=std)
        c.check(c.attn(), p_step=P_STEP_FEW[dtype])


def test_check_rows_counts_a_half_step():
    ref = torch.tensor([1.0], dtype=torch.float64)
    check_rows(torch.tensor([1.0]).bfloat16(), ref, torch.zeros(1, dtype=torch.float64))
    with pytest.raises(AssertionError):
        check_rows(torch.tensor([1.0 + 2.0 ** -7]).bfloat16(), ref, torch.zeros(1, dtype=torch.float64))
