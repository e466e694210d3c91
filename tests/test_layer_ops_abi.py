"""C-ABI checks of the residual norm, the rotating append, the attention with first
tokens in sight and the low-rank adapters that need no GPU: struct layouts, and
every bad argument refused with a message before any HIP call."""
import ctypes
import os
import shutil
import subprocess

import pytest

import busfill as bf
from test_ops_abi import ATTENTION, CACHES, FAKE, attention, cache, refused


@pytest.mark.parametrize("cls,name", [
    (bf.Kv4AppendArgs, "bf_kv4_append_args"), (bf.RmsNormArgs, "bf_rms_norm_args"), (bf.LoraPart, "bf_lora_part"),
    (bf.LoraArgs, "bf_lora_args")])
def test_structs_match_the_header(cls, name, tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "busfill.h"\nint main(void) {\n'
                   f'  printf("%zu\\n", sizeof({name}));\n'
                   + "".join(f'  printf("%zu %zu\\n", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));\n'
                             for f, _ in cls._fields_) + "  return 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run([gcc, "-I", os.path.dirname(bf.HEADER), str(src), "-o", exe], check=True)
    got = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")
    assert int(got[0]) == ctypes.sizeof(cls)
    for line, (f, _) in zip(got[1:], cls._fields_):
        assert tuple(map(int, line.split())) == (getattr(cls, f).offset, getattr(cls, f).size), f


# ------------------------------------------------------------------ attention with first tokens in sight
def test_sinks_refuse():
    L = bf.lib()
    for c, kw, n, needle, st in ([(None, {}, 4, "cache is NULL", bf.ERR_INVALID)]
                                 + [(cache(**k), {}, 4, n, bf.ERR_INVALID) for k, n in CACHES]
                                 + [(cache(), k, 4, n, bf.ERR_INVALID) for k, n in ATTENTION]
                                 + [(cache(), dict(window=64), -1, "sinks=-1", bf.ERR_INVALID),
                                    (cache(), {}, -2 ** 31, "sinks=", bf.ERR_INVALID),
                                    (cache(), dict(max_q=1 << 29), 4, "max_q=", bf.ERR_UNSUPPORTED)]):
        a, cp = attention(**kw), c and ctypes.byref(c)
        refused(lambda: L.bf_kv4_attention_sinks(cp, ctypes.byref(a), n, None), needle, st)
        refused(lambda: L.bf_kv4_attention_sinks_ws(cp, ctypes.byref(a), n, FAKE, 1 << 30, None), needle, st)
        assert L.bf_kv4_attention_sinks_workspace_bytes(cp, ctypes.byref(a), n) == 0
    c = cache()
    refused(lambda: L.bf_kv4_attention_sinks(ctypes.byref(c), None, 4, None), "args is NULL")


def test_sinks_workspace():
    """As without first tokens where there are none or no window; a longer walk of tiles needs more."""
    c = cache(pages=4096)
    a = lambda **kw: attention(ldt=2048, max_kv=131072, **kw)  # noqa: E731
    need = lambda n, **kw: bf.kv4_attention_sinks_workspace_bytes(c, a(**kw), n)  # noqa: E731
    plain = lambda **kw: bf.kv4_attention_workspace_bytes(c, a(**kw))  # noqa: E731
    assert need(0) == plain() == need(1000) and need(0, window=8192) == plain(window=8192) > 0
    assert need(4, window=512) == 0 and need(100000, window=512) > 0
    assert need(2 ** 31 - 1, window=2 ** 31 - 1) > 0
    args, n = a(window=8192), need(64, window=8192)
    ws = lambda p, b: lambda: bf.lib().bf_kv4_attention_sinks_ws(ctypes.byref(c), ctypes.byref(args), 64, p, b, None)  # noqa: E731
    refused(ws(FAKE, n - 1), f"needs {n} bytes")
    refused(ws(FAKE + 16, n), "256-byte")
    refused(ws(None, n), "NULL")


# ------------------------------------------------------------------ append
def append(**kw):
    a = dict(Q=FAKE, ldq=512, Q_out=FAKE + 65536, ldqo=512, K=FAKE, ldk=128, K_out=None, ldko=128, V=FAKE, ldv=128, slots=FAKE,
             positions=FAKE, freq=FAKE, q_heads=8, rot=64, style=0, factor=1.0, T=3)
    a.update(kw)
    return bf.Kv4AppendArgs(*[a[f] for f, _ in bf.Kv4AppendArgs._fields_])


APPEND = [
    (dict(K=None), "NULL", 1), (dict(V=None), "NULL", 1), (dict(slots=None), "NULL", 1), (dict(positions=None), "NULL", 1),
    (dict(freq=None), "NULL", 1), (dict(T=0), "T=0", 1), (dict(T=-3), "T=-3", 1), (dict(ldk=120), "ldk=120", 1),
    (dict(ldv=132), "16-byte", 1), (dict(K=FAKE + 8), "16-byte", 1), (dict(slots=FAKE + 4), "8-byte", 1),
    (dict(positions=FAKE + 4), "8-byte", 1), (dict(freq=FAKE + 2), "4-byte", 1), (dict(rot=0), "rot=0", 1),
    (dict(rot=-16), "rot=-16", 1), (dict(rot=80), "rot=80", 1), (dict(rot=24), "rot=24", 1), (dict(style=2), "style 2", 1),
    (dict(Q=None), "q_heads=8", 1), (dict(Q_out=None), "q_heads=8", 1), (dict(q_heads=0), "q_heads=0", 1),
    (dict(q_heads=-1), "q_heads=-1", 1), (dict(Q=None, Q_out=None), "q_heads=8", 1), (dict(ldq=504), "ld=504 of Q ", 1),
    (dict(ldqo=8), "ld=8 of Q_out", 1), (dict(Q=FAKE + 2), "Q rows", 1), (dict(Q_out=FAKE + 8), "Q_out rows", 1),
    (dict(ldqo=516), "Q_out rows", 1), (dict(K_out=FAKE, ldko=64), "ld=64 of K_out", 1), (dict(K_out=FAKE + 4), "K_out rows", 1),
    (dict(Q_out=FAKE, ldqo=520), "Q_out is Q", 1), (dict(K_out=FAKE, ldko=136), "K_out is K", 1),
    (dict(q_heads=(1 << 20) + 1, ldq=1 << 27, ldqo=1 << 27), "q_heads=1048577", 2), (dict(T=1 << 24), "T=16777216", 2)]


def test_append_refuses():
    L = bf.lib()
    for c, kw, needle, st in ([(None, {}, "cache is NULL", 1)] + [(cache(**k), {}, n, 1) for k, n in CACHES]
                              + [(cache(), *k) for k in APPEND]):
        a, cp = append(**kw), c and ctypes.byref(c)
        refused(lambda: L.bf_kv4_append(cp, ctypes.byref(a), None), needle, st)
    c = cache()
    refused(lambda: L.bf_kv4_append(ctypes.byref(c), None, None), "args is NULL")


# ------------------------------------------------------------------ norm
def norm(**kw):
    a = dict(X=FAKE, xtype=bf.F32, ldx=64, delta=FAKE + 4096, dtype=bf.F16, ldd=64, R=FAKE, ldr=64, weight=FAKE, wtype=bf.F32, offset=0.0,
             eps=1e-6, H=FAKE + 8192, ldh=64, Aq=None, T=3, K=64)
    a.update(kw)
    return bf.RmsNormArgs(*[a[f] for f, _ in bf.RmsNormArgs._fields_])


@pytest.mark.parametrize("kw,needle,status", [
    (dict(X=None), "X is NULL", 1), (dict(H=None), "both NULL", 1), (dict(T=0), "T=0", 1), (dict(K=0), "K=0", 1),
    (dict(T=-1), "T=-1", 1), (dict(xtype=2), "xtype 2", 1), (dict(dtype=-1), "dtype -1", 1), (dict(wtype=3), "wtype 3", 1),
    (dict(ldx=63), "ldx=63", 1), (dict(ldd=1), "ldd=1", 1), (dict(ldr=63, R=FAKE + 64), "ldr=63", 1), (dict(ldh=63), "ldh=63", 1),
    (dict(X=FAKE + 2), "aligned", 1), (dict(delta=FAKE + 1), "aligned", 1), (dict(R=FAKE + 66), "aligned", 1),
    (dict(weight=FAKE + 2), "aligned", 1), (dict(weight=FAKE + 1, wtype=bf.F16), "aligned", 1), (dict(H=FAKE + 1), "aligned", 1),
    (dict(ldr=72), "R is X", 1), (dict(H=FAKE + 4096, ldh=72), "H is delta", 1),
    (dict(H=FAKE + 4096, dtype=bf.F32), "H is delta", 1), (dict(Aq=FAKE, K=40), "multiple of 32", 1),
    (dict(Aq=FAKE + 8), "16-byte", 1), (dict(eps=-1e-9), "eps", 1), (dict(eps=float("nan")), "eps", 1),
    (dict(eps=float("inf")), "eps", 1), (dict(K=32776, ldx=32776, ldd=32776, ldr=32776, ldh=32776), "K=32776", 2),
    (dict(T=1 << 22), "T=4194304", 2)])
def test_norm_refuses(kw, needle, status):
    a = norm(**kw)
    refused(lambda: bf.lib().bf_rms_norm(ctypes.byref(a), None), needle, status)


def test_norm_refuses_null():
    refused(lambda: bf.lib().bf_rms_norm(None, None), "args is NULL")


# ------------------------------------------------------------------ adapters
def lora(slices=((FAKE, FAKE, 64, 0), (FAKE, FAKE, 32, 64)), **kw):
    kept = bf.lora_parts(slices)
    a = dict(X=FAKE, ldx=64, ids=FAKE, scales=None, ranks=None, adapters=4, rank=16, parts=len(slices), part=kept, C=FAKE, ldc=96,
             Y=FAKE + 65536, ldy=96, otype=bf.OUT_F16, T=3, K=64)
    a.update(kw)
    return bf.LoraArgs(*[a[f] for f, _ in bf.LoraArgs._fields_]), kept


LORA = [
    (dict(X=None), "NULL", 1), (dict(ids=None), "NULL", 1), (dict(part=None), "NULL", 1), (dict(C=None), "NULL", 1),
    (dict(Y=None), "NULL", 1), (dict(T=0), "T=0", 1), (dict(adapters=0), "adapters=0", 1), (dict(K=0), "K=0", 1),
    (dict(K=60), "K=60", 1), (dict(rank=0), "rank=0", 1), (dict(rank=12), "rank=12", 1), (dict(rank=-8), "rank=-8", 1),
    (dict(parts=0), "parts=0", 1), (dict(parts=5), "parts=5", 1), (dict(otype=2), "otype 2", 1), (dict(ldx=56), "ld=56 of X", 1),
    (dict(ldx=68), "16-byte", 1), (dict(X=FAKE + 8), "16-byte", 1), (dict(C=FAKE + 1), "aligned", 1), (dict(Y=FAKE + 1), "aligned", 1),
    (dict(C=FAKE + 2, otype=0), "aligned", 1), (dict(ids=FAKE + 2), "4-byte", 1), (dict(scales=FAKE + 1), "4-byte", 1),
    (dict(ranks=FAKE + 2), "4-byte", 1), (dict(Y=FAKE, ldy=104), "Y is C", 1), (dict(ldc=95), "ldc=95", 1), (dict(ldy=95), "ldy=95", 1),
    ([(None, FAKE, 64, 0)], "A or B is NULL", 1), ([(FAKE, None, 64, 0)], "A or B is NULL", 1),
    ([(FAKE + 8, FAKE, 64, 0)], "16-byte", 1), ([(FAKE, FAKE + 4, 64, 0)], "16-byte", 1), ([(FAKE, FAKE, 0, 0)], "N=0", 1),
    ([(FAKE, FAKE, 64, -1)], "at=-1", 1), ([(FAKE, FAKE, 64, 0), (FAKE, FAKE, 8, 63)], "overlap", 1),
    ([(FAKE, FAKE, 8, 40), (FAKE, FAKE, 64, 0)], "overlap", 1), ([(FAKE, FAKE, 64, 33)], "columns 33", 1),
    ([(FAKE, FAKE, 2 ** 31 - 1, 2 ** 31 - 1)], "columns", 1),
    (dict(rank=1032), "rank=1032", 2), (dict(K=(1 << 24) + 8, ldx=1 << 25), "K=16777224", 2),
    (dict(T=(1 << 31) - 1, rank=1024), "workgroups", 2)]


def test_lora_refuses():
    L = bf.lib()
    for what, needle, st in LORA:
        a, kept = lora(**what) if isinstance(what, dict) else lora(what)
        refused(lambda: L.bf_lora(ctypes.byref(a), None), needle, st)
        refused(lambda: L.bf_lora_ws(ctypes.byref(a), FAKE, 1 << 60, None), needle, st)
        assert L.bf_lora_workspace_bytes(ctypes.byref(a)) == 0
    refused(lambda: L.bf_lora(None, None), "args is NULL")
    a, kept = lora([(FAKE, FAKE, (1 << 24) + 1, 0)], ldc=1 << 25, ldy=1 << 25)
    refused(lambda: L.bf_lora(ctypes.byref(a), None), "N=16777217", 2)


def test_lora_workspace():
    L = bf.lib()
    a, kept = lora()
    n = bf.lora_workspace_bytes(a)
    assert n >= 2 * 3 * 16 * 4                                     # the inner sums of both parts
    ws = lambda p, b: lambda: L.bf_lora_ws(ctypes.byref(a), p, b, None)  # noqa: E731
    refused(ws(FAKE, n - 1), f"needs {n} bytes")
    refused(ws(FAKE + 128, n), "256-byte")
    refused(ws(None, n), "NULL")


def test_wrappers_raise():
    c = cache()
    with pytest.raises(bf.BusfillInvalid):
        bf.kv4_append(c, FAKE, FAKE, FAKE, FAKE, None, 1, stream=0)
    with pytest.raises(bf.BusfillInvalid):
        bf.rms_norm(FAKE, 1, 64, xtype=bf.F32, stream=0)
    with pytest.raises(bf.BusfillInvalid):
        bf.lora(FAKE, FAKE, bf.lora_parts([(FAKE, FAKE, 8, 0)]), FAKE, FAKE, T=1, K=7, adapters=1, rank=8, stream=0)
    with pytest.raises(bf.BusfillInvalid):
        bf.kv4_attention_sinks(c, FAKE, FAKE, FAKE, FAKE, FAKE, sinks=-1, S=1, T=1, q_heads=2, max_q=1, max_kv=32, scale=1.0, ldt=1,
                               window=8, stream=0)
