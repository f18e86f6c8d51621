"""The C ABI of shared prefixes and bounded caches: struct layouts, and the status codes of bad arguments (CPU only;
nothing here reaches a device)."""
import ctypes
import os
import shutil
import subprocess

import pytest

from starkv import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, NULL, SHAPE, DTYPE, ALIGN, RANK, WORKSPACE, LIMIT, FORMAT = 0, -1, -2, -3, -4, -5, -6, -7, -8
FAKE = 0x7F0000000000
WS = ctypes.c_void_p(FAKE)
BIG = 1 << 40


def call(name, d, ws=WS, nb=BIG):
    return getattr(L.lib(), name)(ctypes.byref(d), ws, nb, None)


def test_layouts(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    structs = {"starkv_scores_desc": L.ScoresDesc, "starkv_select_desc": L.SelectDesc, "starkv_keep_desc": L.KeepDesc,
               "starkv_prefix_pack_desc": L.PrefixPackDesc, "starkv_prefix_decode_desc": L.PrefixDecodeDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "starkv.h"', "int main(void) {"]
    for c, py in structs.items():
        lines.append(f'printf("{c} . %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "l.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "l"
    subprocess.run([gcc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n"):
        if ln:
            c, f, n = ln.split()
            py = structs[c]
            assert (ctypes.sizeof(py) if f == "." else getattr(py, f).offset) == int(n), ln


def scores(**kw):
    d = L.ScoresDesc(2, 4, 100, L.F32, FAKE, 400, 100, 0, FAKE, 100)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(batch=0)), (SHAPE, dict(n_heads=0)), (SHAPE, dict(seq_len=0)), (LIMIT, dict(n_heads=1025)),
    (LIMIT, dict(batch=65536)), (LIMIT, dict(seq_len=(1 << 24) + 1)), (DTYPE, dict(dtype=L.I8)), (NULL, dict(logits=None)),
    (NULL, dict(scores=None)), (SHAPE, dict(stride_b=-1)), (SHAPE, dict(scores_stride_b=99)), (ALIGN, dict(logits=FAKE + 2)),
    (ALIGN, dict(scores=FAKE + 2)), (LIMIT, dict(batch=60000, n_heads=1024))])
def test_scores_status(want, kw):
    assert call("starkv_attention_scores", scores(**kw)) == want


def test_scores_workspace():
    lib = L.lib()
    assert lib.starkv_attention_scores_workspace_bytes(ctypes.byref(scores())) == 2 * 4 * 8
    assert lib.starkv_attention_scores_workspace_bytes(ctypes.byref(scores(seq_len=4097, scores_stride_b=4097))) == 2 * 4 * 2 * 8
    assert lib.starkv_attention_scores_workspace_bytes(ctypes.byref(scores(batch=0))) == 0
    assert call("starkv_attention_scores", scores(), nb=63) == WORKSPACE
    assert call("starkv_attention_scores", scores(), ws=None) == WORKSPACE
    assert call("starkv_attention_scores", scores(), ws=ctypes.c_void_p(FAKE + 8)) == ALIGN
    assert lib.starkv_attention_scores(None, WS, BIG, None) == NULL


def select(**kw):
    d = L.SelectDesc(2, 100, 50, 4, 10, FAKE, 100, FAKE, 50)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(batch=-1)), (SHAPE, dict(length=-1)), (SHAPE, dict(keep=101)), (SHAPE, dict(sinks=-1)), (SHAPE, dict(recent=47)),
    (SHAPE, dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1)), (LIMIT, dict(length=(1 << 24) + 1)), (LIMIT, dict(batch=65536)),
    (NULL, dict(scores=None)), (NULL, dict(positions=None)), (SHAPE, dict(positions_stride_b=49)), (ALIGN, dict(scores=FAKE + 1)),
    (OK, dict(batch=0)), (OK, dict(keep=0, sinks=0, recent=0))])
def test_select_status(want, kw):
    assert call("starkv_select_positions", select(**kw)) == want


def test_select_workspace():
    lib, long = L.lib(), dict(length=40000 + 14, scores_stride_b=50000)
    assert lib.starkv_select_positions_workspace_bytes(ctypes.byref(select())) == 0
    pieces = 5                                            # of 8192
    want = 3 * 2 * pieces * 2048 * 4 + 2 * 3 * 8
    assert lib.starkv_select_positions_workspace_bytes(ctypes.byref(select(**long))) == want
    assert call("starkv_select_positions", select(**long), nb=want - 1) == WORKSPACE
    assert call("starkv_select_positions", select(**long), ws=None) == WORKSPACE


H = 3


def latents(fmt=L.FMT_DENSE):
    k = L.KLatent()
    keep = [L.int_array([16, 40, 24]), L.i64_array([0, 1600, 5600]), L.i64_array([16, 40, 24]), L.i64_array([0, 2048, 7168])]
    k.n_kv_heads, k.rank, k.head_offset, k.pos_stride, k.bk_head_offset = H, *keep
    k.stride_b, k.format, k.data, k.bk, k.bk_row_stride = 8000, fmt, FAKE, FAKE, 128
    v = L.VLatent()
    v.rank, v.format, v.data, v.stride_b, v.stride_s = 64, L.FMT_DENSE, FAKE, 6400, 64
    return k, v, keep


def keep_desc(fmt=L.FMT_DENSE, k_kw=None, v_kw=None, **kw):
    k, v, refs = latents(fmt)
    for s, more in ((k, k_kw), (v, v_kw)):
        for a, b in (more or {}).items():
            setattr(s, a, b)
    d = L.KeepDesc(2, 100, 50, L.F16, FAKE, 50, k, v, FAKE, 100, None)
    d._refs = refs
    for a, b in kw.items():
        setattr(d, a, b)
    return d


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(batch=0)), (SHAPE, dict(keep=101)), (SHAPE, dict(keep=-1)), (LIMIT, dict(batch=65536)),
    (LIMIT, dict(length=(1 << 24) + 1, keep=1)), (DTYPE, dict(dtype=L.F32)), (NULL, dict(positions=None)), (SHAPE, dict(positions_stride_b=49)),
    (SHAPE, dict(scores_stride_b=99)), (ALIGN, dict(positions=FAKE + 2)), (ALIGN, dict(scores=FAKE + 2)),
    (NULL, dict(k_kw=dict(data=None))), (NULL, dict(v_kw=dict(data=None))), (SHAPE, dict(k_kw=dict(stride_b=0))),
    (SHAPE, dict(v_kw=dict(stride_b=0))), (SHAPE, dict(v_kw=dict(stride_s=63))), (FORMAT, dict(k_kw=dict(format=9))),
    (RANK, dict(v_kw=dict(rank=0))), (NULL, dict(fmt=L.FMT_INT8_SYM)),
    (SHAPE, dict(fmt=L.FMT_INT8_SYM, k_kw=dict(scale=FAKE, scale_stride_b=300, scale_stride_h=0))),
    (SHAPE, dict(fmt=L.FMT_INT8_SYM, k_kw=dict(scale=FAKE, scale_stride_b=0, scale_stride_h=100))),
    (OK, dict(length=0, keep=0))])
def test_keep_status(want, kw):
    d = keep_desc(**kw)
    assert L.lib().starkv_keep_positions(ctypes.byref(d), None) == want


def pack(k_kw=None, v_kw=None, **kw):
    k, v, refs = latents()
    for s, more in ((k, k_kw), (v, v_kw)):
        for a, b in (more or {}).items():
            setattr(s, a, b)
    d = L.PrefixPackDesc(100, L.F16, k, v, 1.0, FAKE, BIG)
    d._refs = refs
    for a, b in kw.items():
        setattr(d, a, b)
    return d


# 2 strips of 64; chunks of 8 ranks 2 + 5 + 3, pairs of chunks 1 + 3 + 2; V padded to 64 columns
PACKED = 256 + 2 * 2 * 10 * 512 + 6 * 4096 + 128 * 64 * 2


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(length=0)), (LIMIT, dict(length=(1 << 24) + 1)), (DTYPE, dict(dtype=L.F32)), (FORMAT, dict(k_kw=dict(format=L.FMT_INT8_SYM))),
    (FORMAT, dict(v_kw=dict(format=L.FMT_INT8_SYM))), (NULL, dict(k_kw=dict(bk=None))), (SHAPE, dict(k_kw=dict(bk_row_stride=127))),
    (NULL, dict(prefix=None)), (WORKSPACE, dict(prefix_bytes=PACKED - 1)), (ALIGN, dict(prefix=FAKE + 16)), (RANK, dict(v_kw=dict(rank=8193, stride_s=8193)))])
def test_pack_status(want, kw):
    d = pack(**kw)
    assert L.lib().starkv_prefix_pack(ctypes.byref(d), None) == want


def test_pack_bytes():
    assert L.lib().starkv_prefix_bytes(ctypes.byref(pack())) == PACKED
    assert L.lib().starkv_prefix_bytes(ctypes.byref(pack(length=0))) == 0


def decode(own=None, **kw):
    k, v, refs = latents()
    o = L.DecodeDesc()
    o.batch, o.n_q_heads, o.head_dim, o.seq_len, o.dtype = 2, 6, 128, 30, L.F16
    o.q, o.q_stride_b, o.q_stride_h, o.k, o.v, o.uv, o.uv_row_stride = FAKE, 768, 128, k, v, FAKE, 64
    o.rope_table, o.rope_max_positions, o.scale, o.out, o.out_stride_b, o.out_stride_h = FAKE, 4096, 0.1, FAKE, 768, 128
    for a, b in (own or {}).items():
        setattr(o.k if a in ("n_kv_heads", "data") else o, a, b)
    turn = (ctypes.c_float * 64)()
    d = L.PrefixDecodeDesc(o, H, 64, 100, refs[0], FAKE, PACKED, turn, turn, FAKE, 30)
    d._more = (refs, turn)
    for a, b in kw.items():
        setattr(d, a, b)
    return d


@pytest.mark.parametrize("want,kw", [
    (SHAPE, dict(length=0)), (SHAPE, dict(n_kv_heads=0)), (LIMIT, dict(n_kv_heads=65)), (RANK, dict(v_rank=0)), (SHAPE, dict(v_rank=63)),
    (SHAPE, dict(n_kv_heads=2)), (NULL, dict(rank=None)), (NULL, dict(prefix=None)), (SHAPE, dict(prefix_bytes=PACKED - 1)),
    (NULL, dict(turn_cos=None)), (ALIGN, dict(prefix=FAKE + 16)), (ALIGN, dict(scores=FAKE + 1)), (SHAPE, dict(scores_stride_b=29)),
    (SHAPE, dict(own=dict(batch=0))), (SHAPE, dict(own=dict(head_dim=64))), (SHAPE, dict(own=dict(n_q_heads=7))), (DTYPE, dict(own=dict(dtype=L.F32))),
    (LIMIT, dict(own=dict(n_q_heads=66))), (NULL, dict(own=dict(q=None))), (NULL, dict(own=dict(uv=None))), (NULL, dict(own=dict(data=None))),
    (SHAPE, dict(own=dict(rope_max_positions=127))), (SHAPE, dict(own=dict(seq_len=-1))), (SHAPE, dict(own=dict(uv_row_stride=63))),
    (DTYPE, dict(own=dict(out_dtype=L.I8))), (LIMIT, dict(own=dict(batch=65536, seq_len=0))), (LIMIT, dict(own=dict(n_q_heads=66, seq_len=0))),
    (SHAPE, dict(own=dict(n_q_heads=7, seq_len=0))), (NULL, dict(own=dict(out=None, seq_len=0))), (DTYPE, dict(own=dict(dtype=L.E4M3, seq_len=0))),
    (SHAPE, dict(own=dict(uv_row_stride=63, seq_len=0))), (SHAPE, dict(own=dict(rope_max_positions=127, seq_len=0)))])
def test_prefix_decode_status(want, kw):
    assert call("starkv_prefix_decode", decode(**kw)) == want


def test_prefix_decode_workspace():
    lib = L.lib()
    need = lib.starkv_prefix_decode_workspace_bytes(ctypes.byref(decode()))
    assert need > 0 and need % 256 == 0
    assert 0 < lib.starkv_prefix_decode_workspace_bytes(ctypes.byref(decode(own=dict(seq_len=0)))) < need
    assert lib.starkv_prefix_decode_workspace_bytes(ctypes.byref(decode(length=0))) == 0
    assert call("starkv_prefix_decode", decode(), nb=need - 1) == WORKSPACE
    assert call("starkv_prefix_decode", decode(), ws=None) == WORKSPACE
    assert call("starkv_prefix_decode", decode(), ws=ctypes.c_void_p(FAKE + 128)) == ALIGN
    assert lib.starkv_prefix_decode(None, WS, BIG, None) == NULL


def test_decode_scores_status():
    d = decode().own
    d._k = latents()
    d.k, d.v = d._k[0], d._k[1]
    f = L.lib().starkv_decode_attention_scores
    assert f(ctypes.byref(d), None, 30, WS, BIG, None) == NULL
    assert f(ctypes.byref(d), ctypes.c_void_p(FAKE + 2), 30, WS, BIG, None) == ALIGN
    assert f(ctypes.byref(d), WS, 29, WS, BIG, None) == SHAPE
    assert f(ctypes.byref(d), WS, 30, WS, 16, None) == WORKSPACE


def test_host_tensors_are_refused():
    import torch
    import starkv
    x = torch.zeros(1, 2, 8)
    k = starkv.KLatentSpec(torch.zeros(1, 1, 8, 16).half(), [16], [0], [16], 128, torch.zeros(1, 16, 128).half(), [0], 128)
    v = torch.zeros(1, 8, 32).half()
    for f in (lambda: starkv.attention_scores(x), lambda: starkv.select_positions(x[0], 1), lambda: starkv.SharedPrefix(k, v),
              lambda: starkv.keep_positions(k, v, torch.zeros(1, 2, dtype=torch.int32), 8)):
        with pytest.raises(starkv.StarKVError):
            f()


def spread(**kw):
    """Two heads of rank 16 and 40 at offsets and pitches of one's own."""
    off, pitch = L.i64_array(kw.pop("off")), L.i64_array(kw.pop("pitch"))
    d = keep_desc(k_kw=dict(n_kv_heads=2, head_offset=off, pos_stride=pitch, stride_b=kw.pop("stride_b")), **kw)
    d._more = (off, pitch)
    return d


@pytest.mark.parametrize("off,pitch,stride_b", [
    ([0, 0], [40, 40], 8000), ([0, 8], [64, 64], 8000), ([0, 56], [64, 64], 8000), ([24, 0], [56, 56], 8000),
    ([0, 1599], [16, 40], 8000), ([3999, 0], [16, 40], 8000), ([0, 16], [56, 56], 5599), ([0, 1600], [16, 40], 5599),
    ([0, 16], [112, 112], 55), ([0, 16], [111, 111], 56), ([0, 640], [64, 64], 1), ([0, 3200], [16, 40], 1599)])
def test_keep_refuses_rows_that_overlap(off, pitch, stride_b):
    d = spread(off=off, pitch=pitch, stride_b=stride_b)
    assert L.lib().starkv_keep_positions(ctypes.byref(d), None) == SHAPE


def test_keep_refuses_more_workgroups_than_a_grid_holds():
    d = keep_desc(batch=65535, v_kw=dict(rank=8192, stride_s=8192, stride_b=819200))
    assert L.lib().starkv_keep_positions(ctypes.byref(d), None) == LIMIT
