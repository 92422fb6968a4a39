"""Host-side refusals of the paged-cache operators and the log probabilities
(CPU): in the front end before the library is reached, and in the C entry points
before any launch."""
from __future__ import annotations

import pytest
import torch

from wavefront_decoding_amd import _lib, ops


def _m(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def _i(*shape):
    return _m(*shape, dtype=torch.int32)


@pytest.fixture
def front(monkeypatch):
    """The front end's checks alone: meta tensors pass as the current device's, the library is out of reach."""
    monkeypatch.setattr(ops, "_need_current", lambda *ts: None)

    def no_library():
        raise AssertionError("validation should have rejected the call before the library is loaded")

    monkeypatch.setattr(_lib, "load", no_library)


def test_host_tensors_are_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    t, pages = torch.zeros(2, 2, 64), torch.zeros(4, 2, 16, 64)
    cu, one, table = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 4).int()
    cos = torch.zeros(8, 32)
    for call in (lambda: ops.attn_paged(t, pages, pages, table, cu, one, kv_len_max=4),
                 lambda: ops.kv_append_paged(t, t, cu, one, table, pages, pages),
                 lambda: ops.qkv_rope_append_paged(t.view(2, 128), cu, one, table, cos, cos, pages, pages, 1, 1, 64),
                 lambda: ops.logprobs(cos)):
        with pytest.raises(_lib.WfdError, match="GPU tensors"):
            call()


def test_page_layout():
    four, three = _m(5, 2, 32, 64), _m(160, 2, 64)
    assert ops.page_layout(four, four) == (2, 64, 32, 32, 5) == ops.page_layout(four, four, 32)
    assert ops.page_layout(three, three, 16) == (2, 64, 1, 16, 10)
    for bad in ((four, four, 16), (three, three, None), (three, three, 0), (three, three, -16), (three, three, 64),
                (_m(5, 2, 1, 64), _m(5, 2, 1, 64), None), (four, three, None), (four, four.float(), None),
                (four.transpose(1, 2), four.transpose(1, 2), None)):
        with pytest.raises(_lib.WfdError):
            ops.page_layout(*bad)


def test_attn_front_end(front):
    base = dict(q=_m(6, 4, 64), k=_m(9, 2, 16, 64), v=_m(9, 2, 16, 64), table=_i(3, 4), cu=_i(4), lens=_i(3), kw={})

    def call(a):
        ops.attn_paged(a["q"], a["k"], a["v"], a["table"], a["cu"], a["lens"], **(dict(kv_len_max=64) | a["kw"]))

    for bad in (dict(q=_m(6, 4, 128)), dict(q=_m(6, 4, 64, dtype=torch.float32)), dict(q=_m(6, 64, 4).transpose(1, 2)),
                dict(q=_m(6, 256)), dict(v=_m(9, 2, 32, 64)), dict(table=_m(3, 4, dtype=torch.int64)),
                dict(table=_i(2, 4)), dict(table=_i(12)), dict(table=_i(4, 3).t()), dict(cu=_m(4, dtype=torch.int64)),
                dict(cu=_i(0)), dict(lens=_i(2)), dict(lens=_m(3, dtype=torch.int64)), dict(lens=_i(6)[::2]),
                dict(kw=dict(kv_len_max=65)), dict(kw=dict(kv_len_max=-1)), dict(kw=dict(q_len_max=-1)),
                dict(kw=dict(window=-1)), dict(kw=dict(sinks=-1)), dict(kw=dict(page_rows=32)),
                dict(kw=dict(kv_len_max=2 ** 31)), dict(kw=dict(out=_m(6, 4, 64, dtype=torch.float32))),
                dict(kw=dict(out=_m(5, 4, 64))),
                dict(q=_m(6, 4, 64, dtype=torch.float16), k=_m(9, 2, 16, 64, dtype=torch.float16),
                     v=_m(9, 2, 16, 64, dtype=torch.float16))):
        with pytest.raises(_lib.WfdError):
            call(base | bad)


def test_append_front_end(front):
    k, pages = _m(6, 2, 64), _m(9, 2, 16, 64)
    cu, lens, table = _i(4), _i(3), _i(3, 4)
    for bad in (dict(k=_m(6, 3, 64)), dict(k=_m(6, 2, 128)), dict(k=_m(5, 2, 64)), dict(k=k.float()),
                dict(k=_m(6, 64, 2).transpose(1, 2)), dict(pages=_m(9, 2, 16, 64, dtype=torch.float32)),
                dict(cu=_i(5)), dict(table=_i(2, 4)), dict(lens=_m(3, dtype=torch.int64))):
        a = dict(k=k, pages=pages, cu=cu, lens=lens, table=table) | bad
        with pytest.raises(_lib.WfdError):
            ops.kv_append_paged(a["k"], k, a["cu"], a["lens"], a["table"], a["pages"], a["pages"])
    cos = _m(16, 32, dtype=torch.float32)
    for bad in (dict(qkv=_m(6, 500)), dict(qkv=_m(6, 512, dtype=torch.float32)), dict(cos=_m(16, 16).float()),
                dict(cos=_m(16, 32)), dict(H=7), dict(Hkv=1), dict(q_out=_m(3, 4, 64)), dict(cu=_i(5))):
        a = dict(qkv=_m(6, 512), cos=cos, H=4, Hkv=2, q_out=None, cu=cu) | bad
        with pytest.raises(_lib.WfdError):
            ops.qkv_rope_append_paged(a["qkv"], a["cu"], lens, table, a["cos"], a["cos"], pages, pages, a["H"],
                                      a["Hkv"], 64, q_out=a["q_out"])


def test_logprobs_front_end(front):
    l, f = _m(4, 50, dtype=torch.float32), torch.float32
    ids = _m(4, dtype=torch.int64)
    for args, kw in (((_m(4, 50, dtype=torch.float16), ids), {}), ((_m(50, 4).t(), ids), {}), ((_m(200), ids), {}),
                     ((l, _i(4)), {}), ((l, ids[:3]), {}), ((l, ids), dict(top=-1)), ((l, ids), dict(top=65)),
                     ((l[:, :5], ids), dict(top=6)), ((l, ids), dict(n=5)), ((l, ids), dict(n=-1)),
                     ((l,), dict(out=_m(4, dtype=f))), ((l, ids), dict(out=_m(3, dtype=f))),
                     ((l, ids), dict(out=_m(4))), ((l,), dict(entropy_out=_m(3, dtype=f))),
                     ((l,), dict(top=2, top_out=_m(4, 1, dtype=f))), ((l,), dict(top=2, top_ids=_i(4, 2))),
                     ((l,), dict(top_out=_m(4, 1, dtype=f)))):
        with pytest.raises(_lib.WfdError):
            ops.logprobs(*args, **kw)


def _attn(lib, *, n=1, nseq=1, H=4, Hkv=2, Dh=64, dtype=1, br=0, ld=4, per=4, pages=9, rows=16, qm=1, km=64, window=0,
          sinks=0, ptr=None):
    return lib.wfd_attn_paged(ptr, ptr, ptr, br, ptr, ld, per, pages, rows, ptr, ptr, nseq, ptr, n, H, Hkv, Dh, dtype,
                              0.1, qm, km, window, sinks, None, 0, None)


def test_c_entry_points_refuse():
    lib = _lib.load()
    for kw, rc in ((dict(nseq=-1), -1), (dict(Hkv=0), -1), (dict(Hkv=3), -1), (dict(ld=3), -1), (dict(per=-1), -1),
                   (dict(rows=8), -1), (dict(rows=24), -1), (dict(rows=0), -1), (dict(rows=-16), -1),
                   (dict(br=32), -1), (dict(br=-1), -1), (dict(Dh=96), -2), (dict(dtype=2), -2),
                   (dict(pages=2 ** 31), -2), (dict(rows=2 ** 24, per=4), -2), (dict(H=8192), -1), (dict(n=-1), -1),
                   (dict(qm=-1), -1), (dict(km=-1), -1), (dict(km=65), -1), (dict(window=-1), -1),
                   (dict(sinks=-1), -1), (dict(H=66), -2), (dict(), -1), (dict(ptr=8), -1),
                   (dict(ptr=16, rows=1024, km=4096), -4)):
        assert _attn(lib, **kw) == rc, kw
        assert b"wfd_attn_paged" in lib.wfd_last_error(), kw
    assert _attn(lib, n=0) == 0 and _attn(lib, nseq=0) == 0

    def rope(n=1, H=4, Hkv=2, Dh=64, ldq=512, rope_rows=8, rows=16, ptr=None):
        return lib.wfd_qkv_rope_append_paged(ptr, ldq, ptr, ptr, 1, ptr, 4, 4, 9, rows, ptr, ptr, rope_rows, ptr, ptr,
                                             ptr, 0, n, H, Hkv, Dh, 1, None)

    for kw in (dict(H=0), dict(ldq=504), dict(ldq=514), dict(rope_rows=0), dict(rows=8), dict(), dict(ptr=8)):
        assert rope(**kw) == -1, kw
    assert rope(Dh=32) == -2 and rope(n=0) == 0

    def append(n=1, ldk=128, rows=16, Dh=64, ptr=None):
        return lib.wfd_kv_append_paged(ptr, ldk, ptr, 128, ptr, ptr, 1, ptr, 4, 4, 9, rows, ptr, ptr, 0, n, 2, Dh, 1,
                                       None)

    for kw in (dict(ldk=120), dict(ldk=132), dict(rows=40), dict(n=-1), dict(), dict(ptr=8)):
        assert append(**kw) == -1, kw
    assert append(Dh=48) == -2 and append(n=0) == 0

    def logp(n=1, V=10, ld=10, top=0, dtype=0, logits=None, out=None, ids=None):
        return lib.wfd_logprobs(logits, ld, ids, out, None, None, None, top, n, V, dtype, None, 0, None)

    for kw in (dict(n=-1), dict(V=0), dict(ld=9), dict(top=-1), dict(top=11), dict(), dict(logits=16, out=16),
               dict(logits=16, top=2)):
        assert logp(**kw) == -1, kw
    assert logp(dtype=3) == -2 and logp(V=100, ld=100, top=65) == -2 and logp(n=0) == 0 and logp(logits=16) == 0
    assert logp(logits=16, out=16, ids=16, V=40000, ld=40000) == -4


def test_appends_refuse_rows_beyond_the_grid():
    """A row is a workgroup of 256 threads, and a launch has fewer than 2^32 of these."""
    lib = _lib.load()
    for n, rc in ((2 ** 24, -2), (2 ** 31 - 1, -2)):
        assert lib.wfd_kv_append_paged(16, 64, 16, 64, 16, 16, 1, 16, 4, 4, 9, 16, 16, 16, 0, n, 1, 64, 1, None) == rc
        assert b"beyond the grid" in lib.wfd_last_error()
        assert lib.wfd_qkv_rope_append_paged(16, 192, 16, 16, 1, 16, 4, 4, 9, 16, 16, 16, 8, 16, 16, 16, 0, n, 1, 1,
                                             64, 1, None) == rc
        assert b"beyond the grid" in lib.wfd_last_error()


def test_workspace_of_parts_that_can_exist():
    """A slot of a part is Dh + 2 numbers. fp32 sequences of many rows are cut into few parts or none, and a row is of a
    sequence of few rows or of one of many, never of both."""
    f32, bf16 = torch.float32, torch.bfloat16
    slot = lambda Dh: (Dh + 2) * 4  # noqa: E731
    need = ops.attn_paged_workspace_bytes
    # one sequence, every tile of it in one part or in few
    assert need(16384, 1, 32, 1, 128, f32, 16384, 16384) <= 10240 * slot(128) + 512
    assert need(4096, 1, 16, 4, 128, f32, 4096, 8192) <= 10240 * slot(128) + 512
    assert need(4096, 1, 16, 4, 128, bf16, 4096, 8192) <= 131072 * slot(128) + 512
    assert need(2000, 1, 64, 64, 64, f32, 2000, 2000, 100, 4) <= 64 * 64 * 5 * slot(64) + 512
    # ragged ticks: per row and head, parts of 512 keys at most
    for H, Hkv in ((16, 16), (16, 4), (32, 8)):
        for rows, seqs, q in ((8192, 256, 512), (8192, 256, 2048), (4096, 64, 300)):
            for dt in (f32, bf16):
                assert need(rows, seqs, H, Hkv, 128, dt, q, 32768) <= rows * H * 64 * slot(128) + 512
    # single tokens under a window: its parts, one more for where it begins, and the sinks'
    assert need(64, 64, 16, 4, 128, bf16, 1, 32768, 4096, 4) <= 64 * 16 * 11 * slot(128) + 512


def test_by_row_refuses_what_the_other_refuses():
    lib = _lib.load()
    for kw, rc in ((dict(nseq=-1), -1), (dict(rows=24), -1), (dict(Dh=96), -2), (dict(dtype=2), -2), (dict(km=65), -1),
                   (dict(H=66), -2), (dict(), -1), (dict(ptr=8), -1), (dict(ptr=16, rows=1024, km=4096), -4)):
        a = dict(n=1, nseq=1, H=4, Hkv=2, Dh=64, dtype=1, ld=4, per=4, pages=9, rows=16, km=64, ptr=None) | kw
        p = a["ptr"]
        assert lib.wfd_attn_paged_by_row(p, p, p, 0, p, a["ld"], a["per"], a["pages"], a["rows"], p, p, a["nseq"], p,
                                         a["n"], a["H"], a["Hkv"], a["Dh"], a["dtype"], 0.1, 1, a["km"], 0, 0, None, 0,
                                         None) == rc, kw
        assert b"wfd_attn_paged_by_row" in lib.wfd_last_error(), kw
    # parts for every row of a prompt, which fp32 sequences of many rows do without
    need = ops.attn_paged_workspace_bytes
    args = (2000, 1, 16, 16, 128, torch.float32, 2000, 2000)
    assert need(*args) < need(*args, by_row=True) <= 2000 * 16 * 4 * 130 * 4 + 512
    assert need(8, 1, 16, 16, 128, torch.bfloat16, 8, 2000) == need(8, 1, 16, 16, 128, torch.bfloat16, 8, 2000, by_row=True)
