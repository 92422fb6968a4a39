"""Host-side refusals of the serving operators (CPU): in the front end before the
library is reached, and in the C entry points before any launch."""
from __future__ import annotations

import pytest
import torch

from wavefront_decoding_amd import _lib, ops


def _m(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def _q(shape=(64, 2, 64), code=torch.int8):
    e = lambda: _m(*shape[:-1], dtype=torch.uint8)  # noqa: E731
    return ops.QuantKV(_m(*shape, dtype=code), _m(*shape, dtype=code), e(), e())


@pytest.fixture
def front(monkeypatch):
    """The front end's checks alone: meta tensors pass as the current device's, the library is out of reach."""
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_need_current", lambda *ts: None)

    def no_library():
        raise AssertionError("validation should have rejected the call before the library is loaded")

    monkeypatch.setattr(_lib, "load", no_library)


def test_host_tensors_are_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    t = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    cache = ops.QuantKV.zeros((8, 2, 64), device="cpu")
    rows = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.kv_append_q(t, t, cache, rows), lambda: ops.kv_read_q(cache, rows),
                 lambda: ops.attn_decode_q(t, cache, rows, rows.int(), kv_len_max=4)):
        with pytest.raises(_lib.WfdError, match="GPU tensors"):
            call()


def test_operands_on_another_device_are_refused(monkeypatch):
    class Fake:
        is_cuda, device = True, torch.device("cuda:1")
        get_device = staticmethod(lambda: 1)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(_lib.WfdError, match="current device is cuda:0"):
        ops._need_current(Fake())


def test_quant_cache_shapes():
    c = ops.QuantKV.zeros((3, 2, 16, 64), code=torch.int8, device="cpu")
    assert (c.Hkv, c.Dh, c.block_rows, c.code) == (2, 64, 16, _lib.INT8) and c.nbytes == 2 * 3 * 2 * 16 * 65
    codes, exps = torch.zeros(4, 2, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)
    for bad in ((codes.bfloat16(), codes.bfloat16(), exps, exps), (codes, codes[:2], exps, exps),
                (codes, codes, exps[:, :1], exps), (codes, codes, exps, exps.int()),
                (codes, codes.view(torch.float8_e4m3fn), exps, exps),
                (codes, codes, torch.zeros(2, 4, dtype=torch.uint8).t(), exps)):
        with pytest.raises(_lib.WfdError):
            ops.QuantKV(*bad)
    with pytest.raises(_lib.WfdError):
        ops.QuantKV.zeros((4, 2, 64), code=torch.bfloat16, device="cpu")


def test_quant_front_end_refusals(front):
    c, rows = _q(), _m(4, dtype=torch.int64)
    k = _m(4, 2, 64)
    for bad in ((_m(4, 3, 64), k, rows), (k, _m(4, 2, 32), rows), (k, _m(5, 2, 64), rows), (k, k.float(), rows),
                (k, k, _m(3, dtype=torch.int64)), (k, k, _m(4, dtype=torch.int32)),
                (_m(4, 64, 2).transpose(1, 2), k, rows)):
        with pytest.raises(_lib.WfdError):
            ops.kv_append_q(bad[0], bad[1], c, bad[2])
    with pytest.raises(_lib.WfdError, match="dtype"):
        ops.kv_read_q(c, rows, dtype=torch.float16)
    with pytest.raises(_lib.WfdError, match="k_out"):
        ops.kv_read_q(c, rows, k_out=_m(3, 2, 64))
    i32 = _m(4, dtype=torch.int32)
    cos = _m(16, 32, dtype=torch.float32)
    for bad in (dict(qkv=_m(4, 500)), dict(pos=rows), dict(cos=_m(16, 16, dtype=torch.float32)),
                dict(H=7), dict(Hkv=1), dict(q_out=_m(3, 4, 64))):
        a = dict(qkv=_m(4, 512), pos=i32, cos=cos, H=4, Hkv=2, q_out=None) | bad
        with pytest.raises(_lib.WfdError):
            ops.qkv_rope_append_q(a["qkv"], a["pos"], a["cos"], a["cos"], rows, c, a["H"], a["Hkv"], 64, a["q_out"])
    q = _m(4, 4, 64)
    for bad in (dict(q=_m(4, 4, 128)), dict(base=i32), dict(lens=rows), dict(lens=_m(3, dtype=torch.int32)),
                dict(m=0), dict(out=_m(4, 4, 64, dtype=torch.float32)), dict(q=_m(4, 64, 4).transpose(1, 2)),
                dict(q=_m(4, 4, 64, dtype=torch.float16), out=_m(4, 4, 64, dtype=torch.float16))):
        a = dict(q=q, base=rows, lens=i32, m=8, out=None) | bad
        with pytest.raises(_lib.WfdError):
            ops.attn_decode_q(a["q"], c, a["base"], a["lens"], kv_len_max=a["m"], out=a["out"])
    with pytest.raises(_lib.WfdError, match="exceeds the cache block"):
        ops.attn_decode_q(q, _q((4, 2, 16, 64)), rows, i32, kv_len_max=17)


def test_quant_entry_points_check_before_launch():
    lib = _lib.load()
    err = lib.wfd_last_error
    app = lambda n=1, Hkv=2, Dh=64, dt=1, code=0, br=0, ld=128: lib.wfd_kv_append_q(  # noqa: E731
        None, ld, None, ld, None, None, None, None, code, br, None, n, Hkv, Dh, dt, None)
    assert app(n=-1) == -1 and app(Hkv=0) == -1 and app(Hkv=70000) == -1 and app(br=-1) == -1 and b"bad shape" in err()
    assert app(Dh=96) == -2 and app(code=2) == -2 and app(dt=2) == -2 and b"dtype" in err()
    assert app(ld=127) == -1 and b"row pitch" in err()
    assert app(n=0) == 0 and app() == -1 and b"null pointer" in err()
    rope = lambda n=1, H=4, S=8, ld=512: lib.wfd_qkv_rope_append_q(  # noqa: E731
        None, ld, None, None, None, S, None, None, None, None, None, None, 0, 0, n, H, 2, 64, 1, None)
    assert rope(H=0) == -1 and rope(S=0) == -1 and rope(ld=511) == -1 and b"ldq=511" in err()
    assert rope(n=0) == 0 and rope() == -1 and b"null pointer" in err()
    read = lambda n=1, dt=1: lib.wfd_kv_read_q(None, None, None, None, 1, 0, None, None, None, n, 2, 64, dt,  # noqa: E731
                                               None)
    assert read(dt=3) == -2 and read(n=0) == 0 and read() == -1
    att = lambda n=1, H=4, Hkv=2, Dh=64, dt=1, m=8, br=0: lib.wfd_attn_decode_q(  # noqa: E731
        None, None, None, None, None, 0, br, None, None, None, n, H, Hkv, Dh, dt, 0.1, m, None, 0, None)
    assert att(H=3) == -1 and att(m=0) == -1 and att(br=4, m=5) == -1 and b"kv_block_rows=4" in err()
    assert att(H=34) == -2 and att(dt=2) == -2 and att(Dh=32) == -2 and att(n=70000) == -2 and b"beyond" in err()
    assert att(n=0) == 0 and att() == -1 and b"null pointer" in err()


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="made-up device addresses: run only where no GPU is "
                    "visible, so a regressed check cannot launch a kernel on them")
def test_quant_alignment_is_checked():
    lib = _lib.load()
    p = [4096] * 4
    assert lib.wfd_kv_append_q(4096 + 8, 128, 4096, 128, *p, 0, 0, 4096, 1, 2, 64, 1, None) == -1
    assert lib.wfd_kv_append_q(4096, 132, 4096, 128, *p, 0, 0, 4096, 1, 2, 64, 1, None) == -1
    assert lib.wfd_kv_append_q(4096, 128, 4096, 128, 4096 + 4, *p[1:], 0, 0, 4096, 1, 2, 64, 1, None) == -1
    assert lib.wfd_qkv_rope_append_q(4096, 512, 4096, 4096 + 4, 4096, 8, 4096, 4096, *p, 0, 0, 1, 4, 2, 64, 1,
                                     None) == -1
    assert lib.wfd_kv_read_q(*p, 0, 0, 4096, 4096 + 2, 4096, 1, 2, 64, 1, None) == -1
    assert lib.wfd_attn_decode_q(4096 + 2, *p, 0, 0, 4096, 4096, 4096, 1, 4, 2, 64, 1, 0.1, 8, 4096, 1 << 20,
                                 None) == -1
    assert b"16-byte aligned" in lib.wfd_last_error()
    assert lib.wfd_attn_decode_q(4096, *p, 0, 0, 4096, 4096, 4096, 1, 4, 2, 64, 1, 0.1, 8, 4096, 16, None) == -4
    assert b"workspace" in lib.wfd_last_error()


# ---------------------------------------------------------------------------
# drawing tokens
# ---------------------------------------------------------------------------
def test_sample_front_end_refusals(front):
    l, u = _m(4, 100, dtype=torch.float32), _m(4, dtype=torch.float32)
    i32, i64 = _m(4, dtype=torch.int32), _m(4, dtype=torch.int64)
    for kw in (dict(logits=_m(4, 100)), dict(logits=l.t()), dict(logits=l[0]), dict(u=u[:3]), dict(u=u.double()),
               dict(temperature=u[:3]), dict(top_k=i64), dict(top_k=u), dict(top_p=i32), dict(min_p=u.double()),
               dict(n=5), dict(n=-1), dict(out=i32), dict(out=i64[:3]), dict(ring=i64), dict(expect=i64),
               dict(accept=i32), dict(expect=i64, accept=i64), dict(temperature=_m(8, dtype=torch.float32)[::2])):
        a = dict(logits=l, u=u) | kw
        with pytest.raises(_lib.WfdError):
            ops.sample(a.pop("logits"), a.pop("u"), **a)


def test_sample_entry_point_checks_before_launch():
    lib = _lib.load()
    call = lambda n=1, V=10, ld=10, ring=None, expect=None: lib.wfd_sample(  # noqa: E731
        None, ld, None, None, None, None, None, None, ring, None, 0, expect, None, n, V, None, 0, None)
    assert call(n=-1) == -1 and call(V=0) == -1 and call(ld=9) == -1 and b"ld=9" in lib.wfd_last_error()
    assert call(V=(1 << 19) + 1, ld=1 << 20) == -2 and b"at most 524288" in lib.wfd_last_error()
    assert call(n=70000) == -2 and call(n=0) == 0 and call() == -1 and b"null pointer" in lib.wfd_last_error()
    ws = lib.wfd_sample_workspace_bytes  # long rows only; as much for each
    assert ws(100, 32768) == 0 and ws(0, 50000) == 0 and ws(3, 1 << 20) == 0
    assert ws(1, 32769) > 8 * 1024 + 8 * 8192 and ws(7, 500000) == 7 * ws(1, 32769)


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="made-up device addresses: run only where no GPU is "
                    "visible, so a regressed check cannot launch a kernel on them")
def test_sample_workspace_is_checked():
    lib = _lib.load()
    call = lambda ws, size: lib.wfd_sample(4096, 50000, 4096, None, None, None, None, 4096, None, None, 0,  # noqa: E731
                                           None, None, 2, 50000, ws, size, None)
    assert call(None, 1 << 30) == -1 and b"null pointer" in lib.wfd_last_error()
    assert call(4096 + 8, 1 << 30) == -1 and b"16-byte aligned" in lib.wfd_last_error()
    assert call(4096, 1000) == -4 and b"workspace 1000 bytes" in lib.wfd_last_error()


def test_sampler_parameters_and_numbers():
    from wavefront_decoding_amd.acceptance import SeededSampler
    from wavefront_decoding_amd.policy import SampledPolicy, SsdPolicy

    for bad in (dict(temperature=-0.1), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1),
                dict(min_p=1.5), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            SeededSampler(0, **bad)
        with pytest.raises(ValueError):
            SampledPolicy(8, 2, **bad)
    with pytest.raises(ValueError):
        SsdPolicy(8, 2, mode="sample")
    with pytest.raises(ValueError):
        SampledPolicy(8, 2, mode="greedy")
    a, b, c = SeededSampler(3), SeededSampler(3), SeededSampler(4)
    at = [0, 1, 4095, 4096, 100000]
    assert [a.uniform(p) for p in at] == [b.uniform(p) for p in reversed(at)][::-1]
    assert all(0.0 <= a.uniform(p) < 1.0 for p in at) and a.uniform(0) != c.uniform(0)
    assert len({a.uniform(p) for p in at}) == len(at)
    made = SampledPolicy(8, 2, sample_seed=5, temperature=0.5, top_k=7).make_sampler()
    assert (made.seed, made.temperature, made.top_k, made.top_p) == (5, 0.5, 7, 1.0)


def test_batch_schedulers_refuse_to_sample():
    """They compare greedy ids, on the device where they can: a sampling policy would decode greedily."""
    from wavefront_decoding_amd.policy import SampledPolicy
    from wavefront_decoding_amd.scheduler_batch import generate_dtv_batch, generate_wavefront_batch

    policy = SampledPolicy(8, 2)
    with pytest.raises(ValueError, match="greedily"):
        generate_wavefront_batch(None, None, 4, policy)
    with pytest.raises(ValueError, match="greedily"):
        generate_dtv_batch(None, None, 4, policy, 2)


# ---------------------------------------------------------------------------
# shared prefixes
# ---------------------------------------------------------------------------
def test_shared_front_end_refusals(front):
    i32, i64 = (lambda n: _m(n, dtype=torch.int32)), (lambda n: _m(n, dtype=torch.int64))
    ok = dict(q=_m(6, 4, 64), k=_m(100, 2, 64), v=_m(100, 2, 64), pb=i64(2), pl=i32(2), gf=i32(3), rb=i64(6), rl=i32(6),
              prefix_len_max=50, kv_len_max=10)
    for bad in (dict(q=_m(6, 4, 128)), dict(q=_m(4, 6, 64).transpose(0, 1)), dict(k=_m(100, 2, 64).float()),
                dict(k=_m(90, 2, 64)), dict(pb=i32(2)), dict(pl=i64(2)), dict(pl=i32(1)), dict(gf=i32(2)),
                dict(gf=i64(3)), dict(rb=i64(5)), dict(rl=i32(5)), dict(rl=i32(12)[::2]), dict(prefix_len_max=-1),
                dict(kv_len_max=-1), dict(group_max=-1), dict(out=_m(5, 4, 64)),
                dict(k=_m(4, 2, 32, 64), v=_m(4, 2, 32, 64)),
                dict(q=_m(6, 4, 64, dtype=torch.float16), k=_m(100, 2, 64, dtype=torch.float16),
                     v=_m(100, 2, 64, dtype=torch.float16))):
        a = ok | bad
        operands = [a.pop(x) for x in ("q", "k", "v", "pb", "pl", "gf", "rb", "rl")]
        with pytest.raises(_lib.WfdError):
            ops.attn_shared(*operands, **a)


def test_shared_entry_point_checks_before_launch():
    lib = _lib.load()
    err = lib.wfd_last_error

    def call(n=2, H=4, Hkv=2, Dh=64, dt=1, ng=1, gm=2, pm=10, om=10, br=0):
        return lib.wfd_attn_shared(None, None, None, br, None, None, None, ng, gm, None, None, None, n, H, Hkv, Dh, dt,
                                   0.1, pm, om, None, 0, None)

    for bad in (dict(n=-1), dict(H=0), dict(H=3), dict(ng=-1), dict(gm=-1), dict(pm=-1), dict(om=-1), dict(br=-1)):
        assert call(**bad) == -1 and b"bad shape" in err(), bad
    assert call(br=8) == -1 and b"exceed a block" in err()
    assert call(dt=2) == -2 and call(Dh=32) == -2 and call(H=34) == -2 and b"G=17" in err()
    assert call(n=0) == 0 and call() == -1 and b"null pointer" in err()
    # the parts: 256 / Hkv chunks at most while they are below 1024 keys, then 1024 keys each; own keys apart
    size = lambda parts: sum(-(-x // 256) * 256 for x in (parts * 64 * 4, parts * 8))  # noqa: E731
    ws = lib.wfd_attn_shared_workspace_bytes
    assert ws(2, 4, 2, 64, 0, 0) == 0 and ws(0, 4, 2, 64, 100, 100) == 0 and ws(2, 4, 2, 64, -1, 0) == 0
    assert ws(2, 4, 2, 64, 128, 0) == size(8) and ws(2, 4, 2, 64, 129, 0) == size(16)
    assert ws(2, 4, 2, 64, 200 * 1024, 0) == size(8 * 200)


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="made-up device addresses: run only where no GPU is "
                    "visible, so a regressed check cannot launch a kernel on them")
def test_shared_alignment_workspace_and_grid_are_checked():
    lib = _lib.load()

    def call(q=4096, ws=4096, size=1 << 30, n=2, ng=1, gm=2, pm=10, om=10):
        return lib.wfd_attn_shared(q, 4096, 4096, 0, 4096, 4096, 4096, ng, gm, 4096, 4096, 4096, n, 4, 2, 64, 1, 0.1,
                                   pm, om, ws, size, None)

    assert call(q=4096 + 2) == -1 and call(ws=4096 + 8) == -1 and b"16-byte aligned" in lib.wfd_last_error()
    assert call(size=16) == -4 and b"workspace" in lib.wfd_last_error()
    assert call(n=70000, size=1 << 60) == -2 and b"beyond the grid" in lib.wfd_last_error()
    assert call(n=60000, gm=60000, ng=60000, pm=1 << 24, size=1 << 60) == -2


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="made-up device addresses: run only where no GPU is "
                    "visible, so a regressed check cannot launch a kernel on them")
def test_quant_calls_past_the_grid_are_refused():
    """2^24 workgroups of 256 threads are more than a launch takes in x."""
    lib = _lib.load()
    p, W = [4096] * 4, 1 << 24
    app = lambda n, dt: lib.wfd_kv_append_q(4096, 128, 4096, 128, *p, 0, 0, 4096, n, 2, 64, dt, None)  # noqa: E731
    read = lambda n: lib.wfd_kv_read_q(*p, 0, 0, 4096, 4096, 4096, n, 2, 64, 1, None)  # noqa: E731
    rope = lambda n: lib.wfd_qkv_rope_append_q(4096, 512, 4096, 4096, 4096, 8, 4096, 4096, *p, 0, 0, n, 4, 2, 64,  # noqa: E731
                                               1, None)
    for call, rows in ((lambda n: app(n, 1), 16), (lambda n: app(n, 0), 8), (read, 8), (rope, 4)):  # rows a workgroup
        assert call(rows * W) == -2 and b"beyond the grid" in lib.wfd_last_error()
        assert call(rows * (W - 1) + 1) == -2


def test_shared_workspace_of_lengths_up_to_the_largest():
    """The parts of bounds next to 2^31 are counted, not wrapped; what the call refuses has none."""
    ws = _lib.load().wfd_attn_shared_workspace_bytes
    size = lambda parts, Dh: sum(-(-x // 256) * 256 for x in (parts * Dh * 4, parts * 8))  # noqa: E731
    top = 2 ** 31 - 1
    for length in (top, top - 127, top - 128, top - 511, top - 1022, top - 1023, top - 1024, top - 2048):
        assert ws(4, 16, 4, 128, length, 0) == size(4 * 16 * -(-length // 1024), 128)
        assert ws(4, 16, 4, 64, 0, length) == size(4 * 16 * -(-length // 512), 64)
    assert ws(65535, 4096, 4096, 128, top, top) == size(65535 * 4096 * (2 ** 21 + 2 ** 22), 128)
    for n, H, Dh in ((65536, 4, 64), (4, 4097, 64), (4, 4, 1 << 20), (top, top, top)):
        assert ws(n, H, H, Dh, top, top) == 0


def test_counts_beyond_32_bits_are_refused_not_cut_off(front, monkeypatch):
    """2^32 + 5 would reach the library as 5, a bound below the lengths."""
    i32, i64 = (lambda n: _m(n, dtype=torch.int32)), (lambda n: _m(n, dtype=torch.int64))
    q, cache = _m(6, 4, 64), _m(100, 2, 64)
    shared = lambda **kw: ops.attn_shared(q, cache, cache, i64(2), i32(2), i32(3), i64(6), i32(6),  # noqa: E731
                                          **(dict(prefix_len_max=50, kv_len_max=10) | kw))
    for n in (2 ** 31, 2 ** 32 + 5):
        for kw in (dict(prefix_len_max=n), dict(kv_len_max=n)):
            with pytest.raises(_lib.WfdError, match="above 2147483647"):
                shared(**kw)
        with pytest.raises(_lib.WfdError, match="above"):
            ops.attn_decode_q(q, _q(), i64(6), i32(6), kv_len_max=n)
    with pytest.raises(_lib.WfdError, match="above 2147482624"):
        ops.attn_decode_q(q, _q(), i64(6), i32(6), kv_len_max=2 ** 31 - 1023)
    u = _m(4, dtype=torch.float32)
    with pytest.raises(_lib.WfdError, match="vocabulary 4294967301"):
        ops.sample(_m(4, 2 ** 32 + 5, dtype=torch.float32), u)
    with pytest.raises(_lib.WfdError, match="rows 4294967301"):
        ops.sample(_m(2 ** 32 + 5, 1, dtype=torch.float32), _m(2 ** 32 + 5, dtype=torch.float32))
    # a group holds at most the call's rows, whatever bound is given
    sent = []

    class Lib:
        wfd_attn_shared_workspace_bytes = staticmethod(lambda *a: 16)
        wfd_attn_shared = staticmethod(lambda *a: sent.append(a) or 0)

    monkeypatch.setattr(_lib, "load", Lib)
    monkeypatch.setattr(ops, "_workspace", lambda need, device: _m(need, dtype=torch.uint8))
    for given, used in ((2 ** 32, 6), (None, 6), (3, 3), (0, 0)):
        shared(group_max=given)
        assert sent[-1][8] == used


def test_quant_attention_counts_whole_splits():
    lib = _lib.load()
    call = lambda m: lib.wfd_attn_decode_q(None, None, None, None, None, 0, 0, None, None, None, 1, 4, 2, 64, 1,  # noqa: E731
                                           0.1, m, None, 0, None)
    for m in (2 ** 31 - 1, 2 ** 31 - 1023):
        assert call(m) == -2 and b"beyond the grid" in lib.wfd_last_error()
    assert call(2 ** 31 - 1024) == -1 and b"null pointer" in lib.wfd_last_error()


def test_quant_cache_follows_its_tensors():
    """Its tensors cannot be exchanged, and ones that were resized or moved in place are used
    where they are, after the checks of a new cache."""
    c = ops.QuantKV.zeros((8, 2, 64), code=torch.int8, device="cpu")
    for name in ("k", "v", "k_exp", "v_exp", "tensors"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name))
    where = lambda: tuple(t.data_ptr() for t in c.tensors)  # noqa: E731
    assert c.pointers() == where()
    c.k.data = torch.zeros(8, 2, 64, dtype=torch.int8)
    c.v_exp.set_(torch.zeros(8, 2, dtype=torch.uint8))
    assert c.pointers() == where()
    for t, shape in zip(c.tensors, ((4096, 4, 64),) * 2 + ((4096, 4),) * 2):
        t.resize_(shape)
    assert c.pointers() == where() and (c.Hkv, c.Dh) == (4, 64)
    c.v.resize_(40960, 4, 64)
    with pytest.raises(_lib.WfdError, match="differ in shape"):
        c.pointers()


@pytest.mark.parametrize("head_major", [True, False])
def test_quant_slots_read_back_only_what_they_hold(monkeypatch, head_major):
    """Ids count from the end below 0, as in the unquantised cache, and rows outside the slots
    never reach the kernel, which trusts them."""
    from wavefront_decoding_amd.kv_cache import BatchStaticKVCache, QuantBatchKVCache

    cache = QuantBatchKVCache(3, 2, 1, 64, 10, torch.bfloat16, "cpu", head_major=head_major)
    plain = BatchStaticKVCache(3, 2, 1, 64, 10, torch.float32, "cpu", head_major=head_major)
    plain.K[:, :, :, 0, 0] = torch.arange(60.0).view(3, 2, 10)  # every row's number
    asked = []

    def read(flat, rows, dtype):
        assert not rows.numel() or 0 <= int(rows.min()) and int(rows.max()) < 60
        asked.append(rows.tolist())
        return rows, rows

    monkeypatch.setattr(ops, "kv_read_q", read)
    for at in (([0, 2], [1, 0], [3, 9]), ([-1, -3], [-1, 1], [0, 4]), ([1], [0], [-1])):
        cache.gather_pack(*at)
        assert asked.pop() == plain.gather_pack(*at)[0][:, 0, 0].tolist()
    for at in (([3], [0], [0]), ([-4], [0], [0]), ([0], [2], [0]), ([0], [-3], [0]), ([0], [0], [10]), ([2], [1], [-2])):
        with pytest.raises(IndexError):
            cache.gather_pack(*at)
    assert not asked


@pytest.mark.parametrize("quant", [False, True])
def test_slots_are_written_only_where_they_are(monkeypatch, quant):
    """Slots and sequences past the cache are an IndexError before any row is written, and
    count from the end below 0."""
    from wavefront_decoding_amd.kv_cache import BatchStaticKVCache, QuantBatchKVCache

    cls = QuantBatchKVCache if quant else BatchStaticKVCache
    cache = cls(3, 2, 1, 64, 10, torch.bfloat16, "cpu")
    wrote = []
    monkeypatch.setattr(ops, "kv_append", lambda k, v, fk, fv, rows: wrote.append(rows.tolist()))
    monkeypatch.setattr(ops, "kv_append_q", lambda k, v, flat, rows: wrote.append(rows.tolist()))
    k, t = torch.zeros(1, 2, 1, 64), torch.zeros(1, 1, 64)
    for slot, b in ((3, 0), (-4, 0), (0, 2), (0, -3)):
        with pytest.raises(IndexError):
            cache.write_prefill(slot, k, k, seq_ids=[b])
        with pytest.raises(IndexError):
            cache.write_tokens([slot], [b], [0], t, t)
    assert not wrote and cache.seqlen == [[0, 0]] * 3
    cache.write_prefill(-1, k, k, seq_ids=[-2])
    cache.write_tokens([-3], [-1], [4], t, t)
    assert wrote == [[40, 41], [14]] and cache.seqlen == [[0, 5], [0, 0], [2, 0]]


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="what is said where no GPU is visible")
def test_host_tensors_are_refused_without_a_gpu():
    t, rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    cache, u = ops.QuantKV.zeros((8, 2, 64), device="cpu"), torch.zeros(2)
    for call in (lambda: ops.kv_append_q(t, t, cache, rows), lambda: ops.kv_read_q(cache, rows),
                 lambda: ops.qkv_rope_append_q(t.view(2, 128), rows.int(), u, u, rows, cache, 2, 2, 64),
                 lambda: ops.attn_decode_q(t, cache, rows, rows.int(), kv_len_max=4), lambda: ops.sample(t[0].float(), u),
                 lambda: ops.attn_shared(t, t, t, rows, rows.int(), rows.int(), rows, rows.int(), prefix_len_max=1,
                                         kv_len_max=1)):
        with pytest.raises(_lib.WfdError, match="GPU tensors"):
            call()


def test_sampler_takes_any_top_k(monkeypatch):
    """More than any vocabulary is off, also past what the operator's 32 bits hold."""
    from wavefront_decoding_amd.acceptance import SeededSampler

    sent = []
    monkeypatch.setattr(ops, "sample", lambda row, u, top_k, **kw: sent.append(top_k.tolist()) or torch.tensor([7]))
    for k, used in ((5, 5), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (10 ** 12, 2 ** 31 - 1)):
        assert SeededSampler(0, top_k=k)(torch.zeros(9), 3) == 7 and sent[-1] == [used]
