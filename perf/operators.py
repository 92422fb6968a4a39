"""Serving operators: an 8-bit slot cache with the attention that reads it,
attention of several answers to one prompt, and the drawing of their tokens.

  listed()          the fixed cases
  draw(rng)         one more case of the same ranges
  prepare(case, s)  inputs and caches, from the seed
  run(state)        one pass: the library's calls (`own`), or the plain form
  work(case)        bytes and operations a pass cannot do without
  exact(case, s)    run()'s outputs from the definitions, in 64 bits

Definitions.

8-bit cache: a row of Dh values x of one kv head is kept as Dh codes and one
exponent byte e + 127: 2^e is the smallest power of two with max|x| <= c 2^e
(c = 448 for e4m3, 127 for int8; e >= -126), a code is x / 2^e rounded once to
nearest, ties to even, and the value it stands for is code * 2^e. A row that is
rotated as it is written is rotated by the float32 cos / sin without rounding
in between.

Attention: softmax(q . k scale) v over the keys that a row attends -- the keys
of its own slot, after those of its group's shared prefix where there is one.

Sampling: with w_j = exp((l_j - max l) / temperature) and the tokens ordered by
logit, largest first, lower index first among equals: the first top_k; of these
the shortest run whose sum of w reaches top_p of theirs; of these the ones with
w_j >= min_p (the first always stays). The token is the lowest kept index whose
running sum of w, in index order over the kept tokens, exceeds u times their
sum. Temperature 0 takes the first token of the order.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CODE_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _ops():
    import __graft_entry__

    __graft_entry__.load_package()
    from wavefront_decoding_amd import ops

    return ops


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # the rows of a single-user wave, rotated and written as they leave the
        # projection, and read back: all latency
        dict(name="qcache_wave8", kind="rope_append", rows=8, H=16, Hkv=16, Dh=128, code="e4m3", dtype="bf16"),
        # the rows of a served batch's tick, grouped heads, odd count
        dict(name="qcache_batch111", kind="rope_append", rows=111, H=16, Hkv=8, Dh=64, code="int8", dtype="bf16"),
        # a long prompt's keys and values written into its slot and read back
        dict(name="qcache_prompt8k", kind="append", rows=8192, H=16, Hkv=16, Dh=128, code="e4m3", dtype="bf16"),
        # one layer's attention of the single-user wave over 8-bit slots
        dict(name="qattn_wave8", kind="qattn", rows=8, H=16, Hkv=16, Dh=128, lo=512, hi=778, code="e4m3",
             dtype="bf16"),
        # the tick of a served batch, ragged prefixes
        dict(name="qattn_batch112", kind="qattn", rows=112, H=16, Hkv=16, Dh=128, lo=128, hi=1200, code="int8",
             dtype="bf16"),
        # long-context decoding with grouped heads
        dict(name="qattn_gqa_32k", kind="qattn", rows=64, H=16, Hkv=4, Dh=128, lo=32700, hi=32768, code="e4m3",
             dtype="bf16"),
        # a few answers to a short prompt, some of them at their first token
        dict(name="shared_4x512", kind="shared", groups=1, rows=4, plo=512, phi=512, lo=0, hi=40, H=16, Hkv=16,
             Dh=128, dtype="bf16"),
        # many answers to one long prompt
        dict(name="shared_64x8k", kind="shared", groups=1, rows=64, plo=8000, phi=8000, lo=1, hi=512, H=16, Hkv=16,
             Dh=128, dtype="bf16"),
        # several prompts with a different number of answers each, grouped heads, long context
        dict(name="shared_gqa_3x32k", kind="shared", groups=3, rows=100, plo=20000, phi=32768, lo=1, hi=300, H=16,
             Hkv=4, Dh=128, dtype="bf16"),
        # one request's next token: temperature, top-k and top-p
        dict(name="sample_1", kind="sample", rows=1, V=32000, std=2.5, mix="both"),
        # a served batch's coda rows, every request with parameters of its own
        dict(name="sample_100", kind="sample", rows=100, V=32000, std=2.5, mix="all"),
        # a large vocabulary whose logits are nearly flat, top-p only
        dict(name="sample_16x128k", kind="sample", rows=16, V=128000, std=1.0, mix="top_p"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["rope_append", "append", "qattn", "qattn", "shared", "shared", "shared", "sample", "sample"])
    H, Hkv, Dh = rng.choice([(16, 16, 128), (16, 16, 128), (16, 4, 128), (4, 4, 64), (4, 2, 64)])
    code = rng.choice(["e4m3", "int8"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if kind == "rope_append":
        return dict(kind=kind, rows=_log_int(rng, 1, 1000), H=H, Hkv=Hkv, Dh=Dh, code=code, dtype=dtype)
    if kind == "append":
        return dict(kind=kind, rows=_log_int(rng, 1, 8192), H=H, Hkv=Hkv, Dh=Dh, code=code, dtype=dtype)
    if kind == "qattn":
        hi = _log_int(rng, 16, 32768)
        rows = _log_int(rng, 1, max(1, min(256, 64 * 32768 * 4 // (hi * Hkv))))
        return dict(kind=kind, rows=rows, H=H, Hkv=Hkv, Dh=Dh, lo=rng.randint(hi // 8, hi), hi=hi, code=code,
                    dtype="bf16" if hi > 4096 else dtype)
    if kind == "shared":
        phi = _log_int(rng, 50, 32768)
        if H == Hkv == 16:
            phi = min(phi, 16384)
        hi = _log_int(rng, 1, 1000)
        groups = _log_int(rng, 1, 6)
        rows = _log_int(rng, 2, 96)
        return dict(kind=kind, groups=min(groups, rows), rows=rows, plo=rng.randint(phi // 2, phi), phi=phi,
                    lo=rng.randint(0, hi), hi=hi, H=H, Hkv=Hkv, Dh=Dh, dtype="bf16" if phi > 2048 else dtype)
    return dict(kind=kind, rows=_log_int(rng, 1, 100), V=_log_int(rng, 1000, 128000),
                std=rng.choice([1.0, 2.0, 3.0]), mix=rng.choice(["plain", "both", "top_p", "all"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed: int, device: str | None = None) -> torch.Generator:
    return torch.Generator(device=device or DEV).manual_seed(seed)


def _randn(g, *shape, dtype, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=g).to(dtype)


def _ints(seed: int, lo: int, hi: int, n: int) -> list[int]:
    return torch.randint(lo, hi + 1, (n,), generator=_gen(seed, "cpu")).tolist()


def _rope(T: int, Dh: int) -> tuple[torch.Tensor, torch.Tensor]:
    theta = 10000.0 ** (-2.0 * torch.arange(Dh // 2, dtype=torch.float64) / Dh)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * theta[None]
    return ang.cos().float().to(DEV), ang.sin().float().to(DEV)


def _lengths(case: dict, seed: int) -> list[int]:
    return _ints(seed + 77, case["lo"], case["hi"], case["rows"])


def _shared_shape(case: dict, seed: int):
    """(first row of every group and the end, prefix lengths, own lengths)."""
    n, ng = case["rows"], case["groups"]
    cuts = sorted(torch.randperm(n - 1, generator=_gen(seed + 79, "cpu"))[: ng - 1].add(1).tolist()) if ng > 1 else []
    return [0] + cuts + [n], _ints(seed + 78, case["plo"], case["phi"], ng), _lengths(case, seed)


def prepare(case: dict, seed: int) -> dict:
    g, kind = _gen(seed), case["kind"]
    st = {"kind": kind, "case": case}
    if kind == "sample":
        n, V = case["rows"], case["V"]
        logits = _randn(g, n, V, dtype=torch.float32, std=case["std"])
        # a grammar forbids part of the vocabulary to every fourth row
        logits[::4, V // 3: V // 2] = -math.inf
        st |= dict(logits=logits, u=torch.rand(n, generator=g, device=DEV))
        return st | _sample_parameters(case, seed)
    n, H, Hkv, Dh, dt = case["rows"], case["H"], case["Hkv"], case["Dh"], DTYPES[case["dtype"]]
    if kind in ("rope_append", "append"):
        # slots of one block of S rows each, rows in no order
        S = max(64, n)
        blocks = 4 if n > 1000 else 16
        row = torch.randperm(blocks * S, generator=_gen(seed + 5, "cpu"))[:n].to(torch.int64).to(DEV)
        st |= dict(flat_row=row, dt=dt)
        if kind == "append":
            st |= dict(k=_randn(g, n, Hkv, Dh, dtype=dt), v=_randn(g, n, Hkv, Dh, dtype=dt))
        else:
            cos, sin = _rope(4096, Dh)
            pos = torch.randint(0, 4096, (n,), generator=_gen(seed + 6, "cpu")).to(torch.int32).to(DEV)
            st |= dict(qkv=_randn(g, n, (H + 2 * Hkv) * Dh, dtype=dt), pos=pos, cos=cos, sin=sin)
        shape = (blocks, Hkv, S, Dh)
        zeros = lambda s, d: torch.zeros(s, dtype=torch.uint8, device=DEV).view(d)  # noqa: E731
        return st | _cache(*(zeros(shape, CODE_DTYPES[case["code"]]) for _ in range(2)),
                           *(zeros(shape[:3], torch.uint8) for _ in range(2)))
    q = _randn(g, n, H, Dh, dtype=dt)
    if kind == "qattn":
        S = case["hi"]
        kq, ke = _codes_of_random(g, (n, Hkv, S, Dh), case["code"])
        vq, ve = _codes_of_random(g, (n, Hkv, S, Dh), case["code"])
        st |= dict(q=q, base=torch.arange(n, dtype=torch.int64, device=DEV) * S,
                   lens=torch.tensor(_lengths(case, seed), dtype=torch.int32, device=DEV))
        return st | _cache(kq, vq, ke, ve)
    first, plen, lens = _shared_shape(case, seed)
    # one block of S rows per answer, and blocks in a row for each prompt
    S, per = max(case["hi"], 1), -(-case["phi"] // max(case["hi"], 1))
    rows = (n + per * case["groups"]) * S
    pbase = [(n + per * j) * S for j in range(case["groups"])]
    dev = lambda x, d: torch.tensor(x, dtype=d, device=DEV)  # noqa: E731
    return st | dict(q=q, k=_randn(g, rows, Hkv, Dh, dtype=dt), v=_randn(g, rows, Hkv, Dh, dtype=dt),
                     first=dev(first, torch.int32), plen=dev(plen, torch.int32), pbase=dev(pbase, torch.int64),
                     base=torch.arange(n, dtype=torch.int64, device=DEV) * S, lens=dev(lens, torch.int32),
                     group_max=max(b - a for a, b in zip(first, first[1:])), host=(first, plen, pbase, lens, S))


def _cache(k, v, k_exp, v_exp) -> dict:
    st = dict(kq=k, vq=v, ke=k_exp, ve=v_exp)
    if own:
        st["cache"] = _ops().QuantKV(k, v, k_exp, v_exp)
    return st


def _codes_of_random(g, shape, code: str):
    """Codes and exponent bytes of a cache of normal values, a block at a time."""
    codes = torch.empty(shape, dtype=CODE_DTYPES[code], device=DEV)
    exps = torch.empty(shape[:3], dtype=torch.uint8, device=DEV)
    for b in range(shape[0]):
        c, e = _quantise(torch.empty(shape[1:], device=DEV).normal_(generator=g), code)
        codes[b], exps[b] = c.to(CODE_DTYPES[code]), (e + 127).to(torch.uint8)
    return codes, exps


def _sample_parameters(case: dict, seed: int) -> dict:
    """Per-request parameters: temperature always; top-k / top-p / min-p by the mix."""
    n, mix, c = case["rows"], case["mix"], _gen(seed + 9, "cpu")
    t = 0.5 + torch.rand(n, generator=c)
    k = torch.randint(1, 200, (n,), generator=c, dtype=torch.int32)
    p = 0.7 + 0.29 * torch.rand(n, generator=c)
    m = 0.1 * torch.rand(n, generator=c)
    if mix == "all":  # some requests greedy, some without one or another limit
        sel = torch.randint(0, 8, (n,), generator=c)
        t[sel == 0] = 0.0
        k[(sel == 1) | (sel == 2)] = 0
        p[(sel == 1) | (sel == 3)] = 1.0
        m[sel != 4] = 0.0
    d = dict(temperature=t.to(DEV), top_k=None, top_p=None, min_p=None)
    if mix in ("both", "all"):
        d["top_k"] = k.to(DEV)
    if mix in ("both", "top_p", "all"):
        d["top_p"] = p.to(DEV)
    if mix == "all":
        d["min_p"] = m.to(DEV)
    return d


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st: dict):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st: dict):
    ops, kind, case = _ops(), st["kind"], st["case"]
    if kind == "rope_append":
        q = ops.qkv_rope_append_q(st["qkv"], st["pos"], st["cos"], st["sin"], st["flat_row"], st["cache"], case["H"],
                                  case["Hkv"], case["Dh"])
        return (q, *ops.kv_read_q(st["cache"], st["flat_row"], dtype=st["dt"]))
    if kind == "append":
        ops.kv_append_q(st["k"], st["v"], st["cache"], st["flat_row"])
        return ops.kv_read_q(st["cache"], st["flat_row"], dtype=st["dt"])
    if kind == "qattn":
        return ops.attn_decode_q(st["q"], st["cache"], st["base"], st["lens"], kv_len_max=case["hi"])
    if kind == "shared":
        return ops.attn_shared(st["q"], st["k"], st["v"], st["pbase"], st["plen"], st["first"], st["base"], st["lens"],
                               prefix_len_max=case["phi"], kv_len_max=case["hi"], group_max=st["group_max"])
    return ops.sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                      min_p=st["min_p"])


def _round_code(v: torch.Tensor, code: str) -> torch.Tensor:
    """v rounded once to the nearest code, ties to even (v: 64 bits, within the codes' range)."""
    if code == "int8":
        return torch.round(v)
    _, e = torch.frexp(v)  # |v| in [2^(e-1), 2^e)
    step = (e - 1).clamp(min=-6).double().sub(3).exp2()
    return torch.round(v / step) * step


def _quantise(x: torch.Tensor, code: str):
    """(codes as 64-bit values, exponents) of rows x (..., Dh)."""
    a = x.abs().amax(-1).double()
    m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1)
    top, bits = (0.875, 9) if code == "e4m3" else (0.9921875, 7)
    e = torch.where(a == 0, -126, torch.where(m <= top, e - bits, e - bits + 1)).clamp(min=-126)
    return _round_code(x.double() * (-e).double().exp2().unsqueeze(-1), code), e


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Interleaved pairs of x (n, heads, Dh) by cos / sin (n, Dh / 2), in 64 bits:
    next to a border between codes, 32 would round twice."""
    c, s, a, b = cos.double()[:, None], sin.double()[:, None], x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)


def _through_cache(st: dict, x: torch.Tensor, codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """Write x (n, Hkv, Dh) at the rows flat_row and read those rows back."""
    case, row = st["case"], st["flat_row"]
    S = codes.shape[2]
    blk, r = row // S, row % S
    c, e = _quantise(x, case["code"])
    codes[blk, :, r] = c.float().to(codes.dtype)
    exps[blk, :, r] = (e + 127).to(torch.uint8)
    return _dequantise(codes[blk, :, r], exps[blk, :, r]).to(st["dt"])


def _dequantise(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    return codes.float() * (exps.float() - 127).exp2().unsqueeze(-1)


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """q (H, Dh) over k / v (Hkv, len, Dh), 32 bits."""
    H, Dh = q.shape
    Hkv = k.shape[0]
    if k.shape[1] == 0:
        return torch.zeros_like(q)
    s = torch.matmul(q.view(Hkv, H // Hkv, Dh), k.transpose(1, 2).contiguous()) / math.sqrt(Dh)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True)).view(H, Dh)


def _run_plain(st: dict):
    kind, case = st["kind"], st["case"]
    if kind == "sample":
        return _sample_plain(st)
    n, H, Hkv, Dh = case["rows"], case["H"], case["Hkv"], case["Dh"]
    if kind == "append":
        return (_through_cache(st, st["k"], st["kq"], st["ke"]), _through_cache(st, st["v"], st["vq"], st["ve"]))
    if kind == "rope_append":
        x = st["qkv"].view(n, H + 2 * Hkv, Dh)
        pos = st["pos"].long()
        y = _rotate(x[:, : H + Hkv], st["cos"][pos], st["sin"][pos])
        return (y[:, :H].to(st["dt"]), _through_cache(st, y[:, H:], st["kq"], st["ke"]),
                _through_cache(st, x[:, H + Hkv:], st["vq"], st["ve"]))
    q, out = st["q"].float(), []
    lens = st["lens"].tolist()
    if kind == "qattn":
        for i, L in enumerate(lens):
            out.append(_attend(q[i], _dequantise(st["kq"][i, :, :L], st["ke"][i, :, :L]),
                               _dequantise(st["vq"][i, :, :L], st["ve"][i, :, :L])))
        return torch.stack(out).to(st["q"].dtype)
    first, plen, pbase, lens, S = st["host"]
    for j in range(case["groups"]):
        for i in range(first[j], first[j + 1]):
            rows = lambda t: torch.cat([t[pbase[j]: pbase[j] + plen[j]], t[i * S: i * S + lens[i]]])  # noqa: E731
            out.append(_attend(q[i], rows(st["k"]).float().transpose(0, 1), rows(st["v"]).float().transpose(0, 1)))
    return torch.stack(out).to(st["q"].dtype)


def _sample_plain(st: dict) -> torch.Tensor:
    """Sorted rows and running sums, in 64 bits: a token is decided by whether a
    long sum lies below or above a border."""
    l, u, t = st["logits"], st["u"].double(), st["temperature"].double()[:, None]
    V = l.shape[1]
    ls, order = torch.sort(l, dim=-1, descending=True, stable=True)
    w = torch.exp((ls.double() - ls[:, :1].double()) / t.clamp(min=1e-300))
    w[:, 0] = 1.0
    rank = torch.arange(V, device=l.device)[None]
    keep = torch.ones_like(l, dtype=torch.bool)
    if st["top_k"] is not None:
        k = st["top_k"].long()[:, None]
        keep &= (rank < k) | (k <= 0)
    if st["top_p"] is not None:
        p = st["top_p"].double()[:, None]
        cum = torch.cumsum(w * keep, -1)
        before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], -1)
        keep &= (before < p * cum[:, -1:]) | (p >= 1.0)
    if st["min_p"] is not None:
        keep &= w >= st["min_p"].double()[:, None]
    keep &= (t > 0) | (rank == 0)
    keep[:, 0] = True
    wk = torch.zeros_like(w).scatter_(1, order, w * keep)
    cum = torch.cumsum(wk, -1)
    return (cum <= u[:, None] * cum[:, -1:]).sum(-1)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    kind, n = case["kind"], case["rows"]
    if kind == "sample":
        return {"bytes": n * (case["V"] * 4 + 8 + 20), "flops": 4.0 * n * case["V"]}
    H, Hkv, Dh, el = case["H"], case["Hkv"], case["Dh"], 2 if case["dtype"] == "bf16" else 4
    if kind in ("append", "rope_append"):
        # values in, codes written and read, values out; the rotated rows' tables and queries too
        b = 2 * n * Hkv * (2 * Dh * el + 2 * (Dh + 1)) + 8 * n
        f = 6.0 * n * Hkv * Dh
        if kind == "rope_append":
            b += 2 * n * H * Dh * el + n * Dh * 4 + 4 * n
            f += 3.0 * n * (H + Hkv) * Dh
        return {"bytes": b, "flops": f}
    mean = (case["lo"] + case["hi"]) / 2
    if kind == "qattn":
        return {"bytes": 2 * n * mean * Hkv * (Dh + 1) + 2 * n * H * Dh * el, "flops": 4.0 * n * mean * H * Dh}
    pre = (case["plo"] + case["phi"]) / 2
    return {"bytes": 2 * (case["groups"] * pre + n * mean) * Hkv * Dh * el + 2 * n * H * Dh * el,
            "flops": 4.0 * n * (pre + mean) * H * Dh}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _exact_values(x: torch.Tensor, code: str) -> torch.Tensor:
    """What rows x (..., Dh) stand for after the 8-bit cache: the codes' own grid
    is laid out and searched (the nearest of the 256 codes, ties to the even one)."""
    if code == "int8":
        grid = torch.arange(-127, 128, dtype=torch.float64, device=x.device)
        c = 127.0
    else:
        pos = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) / 8 * 2.0 ** (e - 7) for e in range(1, 16)
                                                   for m in range(8) if (e, m) != (15, 7)]
        grid = torch.tensor([-p for p in reversed(pos[1:])] + pos, dtype=torch.float64, device=x.device)
        c = 448.0
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((a / c).clamp(min=2.0 ** -126)))
    e = torch.where(a <= c * (e - 1).exp2(), e - 1, e)  # the logarithm may be off by a rounding
    e = torch.where(a > c * e.exp2(), e + 1, e).clamp(min=-126)
    v = x / e.exp2()
    hi = torch.searchsorted(grid, v).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    dl, dh = v - grid[lo], grid[hi] - v
    even = (hi - grid.numel() // 2) % 2 == 0  # code 0 sits in the middle, and codes alternate
    up = (dh < dl) | ((dh == dl) & even)
    return torch.where(up, grid[hi], grid[lo]) * e.exp2()


def _exact_attend(q, keys, values) -> torch.Tensor:
    """q (G, Dh) over lists of key / value pieces (len, Dh) of one kv head."""
    s = torch.cat([q @ k.double().t() for k in keys], -1) / math.sqrt(q.shape[-1])
    if s.shape[-1] == 0:
        return torch.zeros_like(q)
    p = torch.softmax(s, -1)
    out, at = torch.zeros_like(q), 0
    for v in values:
        out += p[:, at: at + v.shape[0]] @ v.double()
        at += v.shape[0]
    return out


def exact(case: dict, seed: int):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "sample":
        return _exact_sample(st)
    n, H, Hkv, Dh = case["rows"], case["H"], case["Hkv"], case["Dh"]
    if kind == "append":
        return _exact_values(st["k"], case["code"]), _exact_values(st["v"], case["code"])
    if kind == "rope_append":
        x = st["qkv"].view(n, H + 2 * Hkv, Dh).double()
        pos = st["pos"].long()
        z = torch.view_as_complex(x[:, : H + Hkv].reshape(n, H + Hkv, Dh // 2, 2).contiguous())
        f = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None]
        y = torch.view_as_real(z * f).reshape(n, H + Hkv, Dh)
        return y[:, :H], _exact_values(y[:, H:], case["code"]), _exact_values(x[:, H + Hkv:], case["code"])
    q, G = st["q"].double(), H // Hkv
    out = torch.zeros(n, H, Dh, dtype=torch.float64, device=DEV)
    if kind == "qattn":
        val = lambda c, e: c.double() * torch.exp2(e.double() - 127)[:, None]  # noqa: E731
        for i, L in enumerate(_lengths(case, seed)):
            for h in range(Hkv):
                out[i, h * G: h * G + G] = _exact_attend(q[i, h * G: h * G + G],
                                                         [val(st["kq"][i, h, :L], st["ke"][i, h, :L])],
                                                         [val(st["vq"][i, h, :L], st["ve"][i, h, :L])])
        return out
    first, plen, pbase, lens, S = st["host"]
    for j in range(case["groups"]):
        for h in range(Hkv):
            pk = st["k"][pbase[j]: pbase[j] + plen[j], h].double()
            pv = st["v"][pbase[j]: pbase[j] + plen[j], h].double()
            for i in range(first[j], first[j + 1]):
                mine = slice(i * S, i * S + lens[i])
                out[i, h * G: h * G + G] = _exact_attend(q[i, h * G: h * G + G], [pk, st["k"][mine, h]],
                                                         [pv, st["v"][mine, h]])
    return out


def _exact_sample(st: dict) -> torch.Tensor:
    """Row by row on the host."""
    host = lambda x: None if x is None else x.cpu().numpy()  # noqa: E731
    l, u, t = host(st["logits"]).astype(np.float64), host(st["u"]), host(st["temperature"])
    k, p, m = host(st["top_k"]), host(st["top_p"]), host(st["min_p"])
    ids = []
    for i in range(l.shape[0]):
        order = np.lexsort((np.arange(l.shape[1]), -l[i]))
        if t[i] == 0:
            ids.append(int(order[0]))
            continue
        if k is not None and k[i] > 0:
            order = order[: int(k[i])]
        w = np.exp((l[i][order] - l[i][order[0]]) / np.float64(t[i]))
        if p is not None and p[i] < 1:
            cum = np.cumsum(w)
            order = order[: int(np.searchsorted(cum, np.float64(p[i]) * cum[-1], side="left")) + 1]
        if m is not None:
            w = w[: len(order)]
            order = order[: max(1, int((w >= np.float64(m[i])).sum()))]
        kept = np.sort(order)
        cum = np.cumsum(np.exp((l[i][kept] - l[i].max()) / np.float64(t[i])))
        ids.append(int(kept[np.searchsorted(cum, np.float64(u[i]) * cum[-1], side="right")]))
    return torch.tensor(ids, device=DEV)
