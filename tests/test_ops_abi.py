"""C-ABI checks of the 4-bit cache, its attention, the routing and the experts'
block that need no GPU: the ctypes structs lie in memory as the header's do, and
every bad argument is refused with a message before any HIP call."""
import ctypes
import os
import shutil
import subprocess

import pytest

import busfill as bf

FAKE = 0x10000   # never dereferenced: every refused call below is refused in validation


@pytest.mark.parametrize("cls,name", [
    (bf.Kv4Cache, "bf_kv4_cache"), (bf.Kv4AttentionArgs, "bf_kv4_attention_args"),
    (bf.MoeRouteArgs, "bf_moe_route_args"), (bf.MoeFfnArgs, "bf_moe_ffn_args")])
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


def refused(call, needle, status=bf.ERR_INVALID):
    assert call() == status
    assert needle in bf.lib().bf_last_error().decode()


# ------------------------------------------------------------------ the cache
@pytest.mark.parametrize("shape,size", [
    ((1, 32, 1, 64), 36 * 64), ((3, 64, 8, 128), 3 * 2 * 8 * 36 * 128), ((2, 96, 5, 96), 2 * 3 * 5 * 36 * 96),
    ((1 << 16, 256, 8, 256), (1 << 22) * 36 * 256),            # more than 2^32 bytes
    ((0, 32, 1, 64), 0), ((1, 0, 1, 64), 0), ((1, 16, 1, 64), 0), ((1, 48, 1, 64), 0), ((1, 32, 0, 64), 0),
    ((1, 32, 1, 80), 0), ((1, 32, 1, 0), 0), ((1, 32, 1, -64), 0), ((-1, 32, 1, 64), 0),
    ((1 << 30, 32, 2, 64), 0), (((1 << 31) - 1, 32, 1, 64), ((1 << 31) - 1) * 36 * 64)])
def test_cache_bytes(shape, size):
    assert bf.kv4_bytes(*shape) == size


CACHES = [(dict(data=None), "cache data is NULL"), (dict(data=FAKE + 128), "256-byte"), (dict(pages=0), "pages=0"),
          (dict(page_size=40), "page_size=40"), (dict(kv_heads=0), "kv_heads=0"), (dict(head_dim=80), "head_dim=80")]


def cache(**kw):
    a = dict(data=FAKE, pages=4, page_size=64, kv_heads=2, head_dim=64)
    a.update(kw)
    return bf.Kv4Cache(a["data"], a["pages"], a["page_size"], a["kv_heads"], a["head_dim"])


def rows(name, c, **kw):
    a = dict(K=FAKE, ldk=128, V=FAKE, ldv=128, slots=FAKE, T=3)
    a.update(kw)
    order = ("K", "ldk", "V", "ldv", "slots", "T") if name == "bf_kv4_store" else ("slots", "K", "ldk", "V", "ldv", "T")
    return lambda: getattr(bf.lib(), name)(c and ctypes.byref(c), *[a[n] for n in order], None)


@pytest.mark.parametrize("name", ["bf_kv4_store", "bf_kv4_load"])
def test_store_and_load_refuse(name):
    refused(rows(name, None), "cache is NULL")
    for kw, needle in CACHES:
        refused(rows(name, cache(**kw)), needle)
    for kw, needle in [(dict(K=None), "NULL"), (dict(V=None), "NULL"), (dict(slots=None), "NULL"), (dict(T=0), "T=0"),
                       (dict(T=-1), "T=-1"), (dict(ldk=127), "ldk=127"), (dict(ldv=64), "ldv=64"),
                       (dict(ldk=132), "16-byte"), (dict(ldv=129), "16-byte"), (dict(K=FAKE + 8), "16-byte"),
                       (dict(V=FAKE + 2), "16-byte"), (dict(slots=FAKE + 4), "8-byte")]:
        refused(rows(name, cache(), **kw), needle)
    refused(rows(name, cache(kv_heads=65536), ldk=1 << 23, ldv=1 << 23), "kv_heads=65536", bf.ERR_UNSUPPORTED)


# ------------------------------------------------------------------ attention
def attention(**kw):
    a = dict(Q=FAKE, O=FAKE, q_start=FAKE, kv_len=FAKE, page_table=FAKE, S=2, T=2, q_heads=8, max_q=1, max_kv=200,
             scale=0.125, ldq=512, ldo=512, ldt=4, causal=True, window=0, otype=bf.OUT_F32, lse=None)
    a.update(kw)
    v = {n: a.pop(n) for n in ("Q", "O", "q_start", "kv_len", "page_table")}
    return bf.kv4_attention_args(cache(), *v.values(), **a)


ATTENTION = [
    (dict(Q=None), "NULL"), (dict(O=None), "NULL"), (dict(q_start=None), "NULL"), (dict(kv_len=None), "NULL"),
    (dict(page_table=None), "NULL"), (dict(S=0), "S=0"), (dict(T=0), "T=0"), (dict(max_q=0), "max_q=0"),
    (dict(max_kv=-1), "max_kv=-1"), (dict(ldt=0, max_kv=0), "ldt=0"), (dict(q_heads=0), "q_heads=0"),
    (dict(q_heads=7), "q_heads=7"), (dict(ldq=511), "ldq=511"), (dict(ldo=100), "ldo=100"), (dict(ldq=516), "16-byte"),
    (dict(Q=FAKE + 8), "16-byte"), (dict(otype=2), "otype 2"), (dict(O=FAKE + 2), "O is not aligned"),
    (dict(O=FAKE + 1, otype=bf.OUT_F16), "O is not aligned"), (dict(lse=FAKE + 2), "4-byte"),
    (dict(q_start=FAKE + 1), "4-byte"), (dict(kv_len=FAKE + 2), "4-byte"), (dict(page_table=FAKE + 3), "4-byte"),
    (dict(max_kv=257), "max_kv=257"), (dict(window=-1), "window=-1"), (dict(window=8, causal=False), "window=8"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=-3.2e38), "scale")]


def test_attention_refuses():
    L = bf.lib()
    for c, kw, needle, st in ([(None, {}, "cache is NULL", bf.ERR_INVALID)]
                              + [(cache(**k), {}, n, bf.ERR_INVALID) for k, n in CACHES]
                              + [(cache(), k, n, bf.ERR_INVALID) for k, n in ATTENTION]
                              + [(cache(), dict(max_q=1 << 29), "max_q=", bf.ERR_UNSUPPORTED),
                                 (cache(), dict(ldt=1 << 26, max_kv=(1 << 31) - 1), "max_kv=", bf.ERR_UNSUPPORTED),
                                 (cache(), dict(S=1 << 30, T=(1 << 31) - 1, max_q=12), "workgroups", bf.ERR_UNSUPPORTED)]):
        a = attention(**kw)
        cp = c and ctypes.byref(c)
        refused(lambda: L.bf_kv4_attention(cp, ctypes.byref(a), None), needle, st)
        refused(lambda: L.bf_kv4_attention_ws(cp, ctypes.byref(a), FAKE, 1 << 30, None), needle, st)
        assert L.bf_kv4_attention_workspace_bytes(cp, ctypes.byref(a)) == 0
    c = cache()
    refused(lambda: L.bf_kv4_attention(ctypes.byref(c), None, None), "args is NULL")


def test_attention_workspace():
    """None where a workgroup sees all of a sequence (a window's span counts, not the cache's); the bytes asked for
    are those the call wants; an unaligned or missing workspace is refused."""
    L, c = bf.lib(), cache(pages=4096)
    need = lambda **kw: bf.kv4_attention_workspace_bytes(c, attention(ldt=2048, **kw))
    assert need(max_kv=1024) == 0 and need(max_kv=0) == 0
    long_ = need(max_kv=131072)
    assert long_ > 0 and need(max_kv=131072, window=512) == 0
    assert need(max_kv=131072, S=64, T=4096, max_q=64) == 0    # rows enough to fill the chip: no chunks
    a = attention(ldt=2048, max_kv=131072)
    ws = lambda p, n: lambda: L.bf_kv4_attention_ws(ctypes.byref(c), ctypes.byref(a), p, n, None)
    refused(ws(FAKE, long_ - 1), f"needs {long_} bytes")
    refused(ws(FAKE + 16, long_), "256-byte")
    refused(ws(None, long_), "NULL")


# ------------------------------------------------------------------ routing
def route(**kw):
    a = dict(logits=FAKE, ltype=bf.LOGITS_F32, ldl=64, bias=None, ids=FAKE, weights=FAKE, T=3, E=64, k=8,
             score=bf.SCORE_SOFTMAX, groups=1, top_groups=1, renorm=1, factor=1.0)
    a.update(kw)
    return bf.MoeRouteArgs(*[a[f] for f, _ in bf.MoeRouteArgs._fields_])


@pytest.mark.parametrize("kw,needle,status", [
    (dict(logits=None), "NULL", 1), (dict(ids=None), "NULL", 1), (dict(weights=None), "NULL", 1),
    (dict(ltype=2), "ltype 2", 1), (dict(score=-1), "score -1", 1), (dict(T=0), "T=0", 1), (dict(E=0), "E=0", 1),
    (dict(k=0), "k=0", 1), (dict(ldl=63), "ldl=63", 1), (dict(groups=0), "groups=0", 1), (dict(groups=7), "groups=7", 1),
    (dict(groups=8, top_groups=0), "top_groups=0", 1), (dict(groups=8, top_groups=9), "top_groups=9", 1),
    (dict(groups=8, top_groups=1, k=9), "only 8", 1), (dict(k=65), "only 64", 1), (dict(logits=FAKE + 2), "aligned", 1),
    (dict(logits=FAKE + 1, ltype=bf.LOGITS_F16), "aligned", 1), (dict(bias=FAKE + 2), "aligned", 1),
    (dict(ids=FAKE + 1), "aligned", 1), (dict(weights=FAKE + 2), "aligned", 1),
    (dict(E=1025, ldl=1025), "E=1025", 2), (dict(E=128, ldl=128, k=65), "k=65", 2),
    (dict(E=130, ldl=130, groups=65, top_groups=8), "groups=65", 2)])
def test_route_refuses(kw, needle, status):
    a = route(**kw)
    refused(lambda: bf.lib().bf_moe_route(ctypes.byref(a), None), needle, status)


def test_route_refuses_null():
    refused(lambda: bf.lib().bf_moe_route(None, None), "args is NULL")


# ------------------------------------------------------------------ the experts' block
def experts(qtype=bf.Q4_K, **kw):
    aux = FAKE if qtype == bf.Q4_0_PLANES else None
    a = dict(gate=(FAKE, aux), up=(FAKE, aux), down=(FAKE, aux), A=FAKE, ids=FAKE, weights=FAKE, C=FAKE, T=4, K=512, F=256,
             N=128, E=8, k=2)
    a.update(kw)
    v = [a.pop(n) for n in ("gate", "up", "down", "A", "ids", "weights", "C")]
    return bf.moe_ffn_args(qtype, *v, **a)


EXPERTS = [
    (dict(qtype=5), "qtype", 1), (dict(T=0), "T=0", 1), (dict(E=0), "E=0", 1), (dict(k=0), "k=0", 1),
    (dict(gate=(None, None)), "W is NULL", 1), (dict(up=(None, None)), "W is NULL", 1),
    (dict(down=(None, None)), "W is NULL", 1), (dict(down=(FAKE, FAKE)), "must be NULL", 1),
    (dict(qtype=bf.Q4_0_PLANES, up=(FAKE, None)), "W_aux", 1), (dict(K=500), "multiple", 1),
    (dict(K=512 + 32), "256", 1), (dict(F=256 + 32), "256", 1), (dict(qtype=bf.Q4_0, F=100), "32", 1),
    (dict(N=0), "N=0", 1), (dict(F=0), "0", 1), (dict(lda=511), "lda=511", 1), (dict(ldc=127), "ldc=127", 1),
    (dict(A=None), "NULL", 1), (dict(C=None), "NULL", 1), (dict(ids=None), "NULL", 1), (dict(weights=None), "NULL", 1),
    (dict(ids=FAKE + 2), "4-byte", 1), (dict(weights=FAKE + 1), "4-byte", 1), (dict(A=FAKE + 1), "aligned", 1),
    (dict(C=FAKE + 2), "aligned", 1), (dict(otype=3), "otype", 1), (dict(E=4097), "E=4097", 2),
    (dict(T=1 << 24, k=2), "T * k", 2), (dict(E=4096, F=1 << 20), "F=1048576", 2), (dict(E=4096, N=1 << 20), "N=1048576", 2),
    (dict(N=(1 << 24) + 1, E=1), "N=16777217", 2), (dict(F=(1 << 24) + 256, E=1), "F=16777472", 2),
    (dict(A=FAKE + 2), "Q4_K", 2), (dict(lda=516), "lda=516", 2), (dict(gate=(FAKE + 4, None)), "Q4_K", 2)]


def test_experts_refuse():
    L = bf.lib()
    for kw, needle, st in EXPERTS:
        a = experts(**kw)
        refused(lambda: L.bf_moe_ffn(ctypes.byref(a), None), needle, st)
        refused(lambda: L.bf_moe_ffn_ws(ctypes.byref(a), FAKE, 1 << 40, None), needle, st)
        assert L.bf_moe_ffn_workspace_bytes(ctypes.byref(a)) == 0
    refused(lambda: L.bf_moe_ffn(None, None), "args is NULL")


@pytest.mark.parametrize("qtype", [bf.Q4_0, bf.Q4_0_PLANES, bf.Q4_K])
def test_experts_workspace(qtype):
    L, a = bf.lib(), experts(qtype)
    need = bf.moe_ffn_workspace_bytes(a)
    assert need >= 8 * (256 * 2 + 128 * 4)                     # h and y of every slot
    assert bf.moe_ffn_workspace_bytes(experts(qtype, otype=bf.OUT_F16)) == need
    many = [bf.moe_ffn_workspace_bytes(experts(qtype, T=400, otype=o)) for o in (bf.OUT_F32, bf.OUT_F16)]
    assert many[1] < many[0]                                   # (y in fp16)
    assert bf.moe_ffn_workspace_bytes(experts(qtype, T=4000)) >= 8000 * (256 * 2 + 128 * 4)
    ws = lambda p, n: lambda: L.bf_moe_ffn_ws(ctypes.byref(a), p, n, None)
    refused(ws(FAKE, need - 1), f"needs {need} bytes")
    refused(ws(FAKE + 128, need), "256-byte")
    refused(ws(None, need), "NULL")


def test_wrappers_raise():
    c = cache()
    with pytest.raises(bf.BusfillInvalid):
        bf.kv4_store(c, FAKE, FAKE, FAKE, 0, stream=0)
    with pytest.raises(bf.BusfillInvalid):
        bf.kv4_load(c, None, FAKE, FAKE, 1, stream=0)
    with pytest.raises(bf.BusfillInvalid):
        bf.kv4_attention(c, FAKE, FAKE, FAKE, FAKE, None, S=1, T=1, q_heads=2, max_q=1, max_kv=32, scale=1.0, ldt=1, stream=0)
    with pytest.raises(bf.BusfillInvalid):
        bf.moe_route(FAKE, FAKE, FAKE, 1, 8, 9, ltype=bf.LOGITS_F32, stream=0)
    with pytest.raises(bf.BusfillError):
        bf.moe_ffn(bf.Q4_K, (FAKE, None), (FAKE, None), (FAKE, None), FAKE, FAKE, FAKE, FAKE, T=1, K=256, F=256, N=16, E=5000,
                   k=1, stream=0)
