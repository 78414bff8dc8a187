"""The calls on heads and a paged cache on the CPU (no GPU): what they refuse,
and what reaches the library."""
import os
import shutil
import struct
import subprocess

import pytest
import torch

from adapterslotsplusplus_amd import _lib, engine as engine_mod
from adapterslotsplusplus_amd.engine import WarpPipeEngine
from adapterslotsplusplus_amd.rotary import Rotary
from tests.test_engine_args_host import RecordingLib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, E4 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture
def eng(monkeypatch):
    """An engine over CPU tensors (device index -1) and the recording library."""
    monkeypatch.setattr(engine_mod, "_raw_stream", lambda dev: 0)
    e = WarpPipeEngine.__new__(WarpPipeEngine)
    e._lib, e._handle, e._dev_index, e._ranks = RecordingLib(), None, -1, {8: True}
    return e


def rows(T=3, heads=4, dim=32, dtype=BF):
    return torch.zeros(T, heads, dim, dtype=dtype)


def pages(n=2, size=16, heads=2, dim=32, dtype=BF):
    return torch.zeros(n, size, heads, dim, dtype=torch.uint8).view(dtype) if dtype == E4 else torch.zeros(n, size, heads, dim, dtype=dtype)


def test_structs_are_the_headers(tmp_path):
    """Their sizes and the fields' places, by a C compiler."""
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not found")
    src = tmp_path / "sizes.c"
    src.write_text('#include "warppipe_mi355x.h"\n#include <stddef.h>\n#include <stdio.h>\nint main(void) {\n'
                   ' printf("%zu %zu %zu %zu %zu %zu %zu %zu %zu %zu\\n", sizeof(wp_head_rows), offsetof(wp_head_rows, heads),'
                   " sizeof(wp_rotation), offsetof(wp_rotation, factor), sizeof(wp_pages), offsetof(wp_pages, k_scale_strides),"
                   " offsetof(wp_pages, e4m3), sizeof(wp_sequences), offsetof(wp_sequences, row_stride), offsetof(wp_sequences, n_seq));\n"
                   " return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run([gcc, "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    e = engine_mod
    assert got == [e._ROWS.size, e._ROWS.size - 8, e._ROTATION.size, e._ROTATION.size - 4, e._PAGES.size, 32 + 6 * 8, e._PAGES.size - 4,
                   e._SEQUENCES.size, 24, e._SEQUENCES.size - 4]


def test_null_arguments_are_errors_not_crashes():
    lib = _lib.load()
    assert lib.wp_rotate_heads(None, None, None, 1e-6, None, 1, 64, 1, None) == _lib.WP_ERR_INVALID
    assert lib.wp_rotate_into_cache(None, None, None, None, 1e-6, None, None, None, 0, 1, 1, None) == _lib.WP_ERR_INVALID
    assert lib.wp_write_cache(None, None, None, None, None, 0, 1, 1, None) == _lib.WP_ERR_INVALID
    assert lib.wp_read_cache(None, None, None, None, None, 0, 1, 1, None) == _lib.WP_ERR_INVALID
    assert lib.wp_paged_attention(None, None, None, None, None, 1, 1.0, 0, 0, 1, None) == _lib.WP_ERR_INVALID
    with pytest.raises(RuntimeError, match="engine is NULL"):
        _lib.check(lib.wp_paged_attention(None, None, None, None, None, 1, 1.0, 0, 0, 1, None), "paged_attention")


def test_views_reach_the_library_as_they_are(eng):
    qkv = torch.zeros(5, 8, 32, dtype=BF)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    turn = Rotary(16, interleaved=True, device="cpu")
    at = torch.arange(5)
    kp, vp = pages().transpose(1, 2).contiguous().transpose(1, 2), pages()
    out = eng.rotate_into_cache(q, k, v, at, turn, kp, vp, at.int(), q_out=q)
    name, a = eng._lib.calls[-1]
    assert name == "wp_rotate_into_cache" and out is q
    qr, kr, vr, eps, rot, cache, slots, wide, T, dt = a[1:11]
    assert struct.unpack("3q4q2i", qr) == (q.data_ptr(), q.data_ptr(), 0, 256, 32, 256, 32, 4, 0)
    assert struct.unpack("3q4q2i", kr)[:1] + struct.unpack("3q4q2i", kr)[3:5] == (k.data_ptr(), 256, 32)
    assert struct.unpack("3q4q2i", vr)[0] == v.data_ptr()
    assert struct.unpack("2q3if", rot) == (turn.turns.data_ptr(), at.data_ptr(), 1, 16, 1, 1.0)
    c = struct.unpack("4q6q6qq4i", cache)
    assert c[:2] == (kp.data_ptr(), vp.data_ptr()) and c[4:10] == (1024, 32, 512, 1024, 64, 32) and c[16:] == (2, 16, 2, 32, 0)
    assert (slots, wide, T, dt) == (a[7], 0, 5, 1) and eps == 1e-6


def test_rotate_heads_refuses(eng):
    q, k, at, turn = rows(), rows(heads=2), torch.arange(3), Rotary(32, device="cpu")
    f = eng.rotate_heads
    for bad, message in ((lambda: f(q.float(), k, at, turn), "fp16 or bf16"), (lambda: f(q, k.half(), at, turn), "k must be"),
                         (lambda: f(q, k[:2], at, turn), "3 tokens, k has 2"), (lambda: f(q, k, at[:2], turn), "positions"),
                         (lambda: f(q, k, at.float(), turn), "positions"), (lambda: f(q, k, None, turn), "needs positions"),
                         (lambda: f(q.transpose(1, 2), k, at, turn), "contiguous"), (lambda: f(q[0], k, at, turn), "tokens, heads"),
                         (lambda: f(q, k, at, turn, q_norm=torch.ones(32)), "q_norm"), (lambda: f(q, k, at, turn, k_norm=torch.ones(16, dtype=BF)), "k_norm"),
                         (lambda: f(q, k, at, turn, q_out=q[:, :2]), "q_out must be")):
        with pytest.raises(RuntimeError, match=message):
            bad()
    assert not eng._lib.calls


def test_cache_calls_refuse(eng):
    k, v, kp, vp, at = rows(heads=2), rows(heads=2), pages(), pages(), torch.arange(3)
    k8, v8, s8 = pages(dtype=E4), pages(dtype=E4), torch.zeros(2, 16, 2, dtype=torch.uint8)
    for f in (eng.write_cache, lambda k, v, *a, **kw: eng.rotate_into_cache(None, k, v, None, None, *a, **kw)):
        for bad, message in ((lambda: f(k, v[:2], kp, vp, at), "as many tokens"), (lambda: f(rows(), v, kp, vp, at), "k and v must be"),
                             (lambda: f(k.half(), v.half(), kp, vp, at), "pages must be"), (lambda: f(k, v, kp, vp[:1], at), "one dtype"),
                             (lambda: f(k, v, kp, vp, at[:2]), "slots"), (lambda: f(k, v, kp, vp, at.float()), "slots"),
                             (lambda: f(k, v, kp, vp, at, k_scales=s8, v_scales=s8), "scales belong"), (lambda: f(k, v, k8, v8, at), "need k_scales"),
                             (lambda: f(k, v, k8, v8, at, k_scales=s8, v_scales=s8[:1]), "v_scales must be"),
                             (lambda: f(k, v, kp[0], vp[0], at), "pages, page_size")):
            with pytest.raises(RuntimeError, match=message):
                bad()
    for bad, message in ((lambda: eng.read_cache(kp, vp, at[:, None]), "slots"), (lambda: eng.read_cache(kp, vp, at, dtype=torch.float16), "pages must be"),
                         (lambda: eng.read_cache(k8, v8, at, s8, s8, dtype=torch.float32), "fp16 or bf16")):
        with pytest.raises(RuntimeError, match=message):
            bad()
    assert not eng._lib.calls


def test_paged_attention_refuses(eng):
    q, kp, vp = rows(), pages(), pages()
    t, cu, n = torch.zeros(2, 2, dtype=torch.int32), torch.tensor([0, 1, 3], dtype=torch.int32), torch.tensor([4, 9], dtype=torch.int32)
    f = eng.paged_attention
    for bad, message in ((lambda: f(q.float(), kp, vp, t, cu, n), "fp16 or bf16"), (lambda: f(q.half(), kp, vp, t, cu, n), "pages must be"),
                         (lambda: f(q[..., :16], kp, vp, t, cu, n), "heads, 32"), (lambda: f(q, kp, vp, t.long(), cu, n), "block_table must be int32"),
                         (lambda: f(q, kp, vp, t, cu.long(), n), "cu_seqlens_q must be int32"), (lambda: f(q, kp, vp, t, cu[:2], n), "cu_seqlens_q"),
                         (lambda: f(q, kp, vp, t[:1], cu, n), "block_table must be"), (lambda: f(q, kp, vp, t.t().contiguous().t(), cu, n), "unit column"),
                         (lambda: f(q, kp, vp, t, cu, n, out=q[:2]), "out must be"), (lambda: f(q, kp, vp, t, cu, n, out=q.half()), "out must be")):
        with pytest.raises(RuntimeError, match=message):
            bad()
    assert not eng._lib.calls
    f(q, kp, vp, t, cu, n, window=5, sinks=2)
    name, a = eng._lib.calls[-1]
    assert name == "wp_paged_attention" and struct.unpack("3qq2i", a[4])[3:] == (2, 2, 2) and a[5] == 3 and a[7:9] == (5, 2)
