"""What the entry points of 8-bit caches in blocks (include/ns_kv8.h) refuse, through the C ABI and before any GPU is touched; their
scratch; the Python wrappers' own checks; the C++ table. Arguments that nothing is wrong with end at the null handle."""
import ctypes as C
import os
import re
import subprocess
import types

import numpy as np
import pytest

from kv8_ref import E4, E4M3, HELD, INT8, MOST, Cache, encode, scale_of, values
from nextsycl_amd import Error, library_path
from nextsycl_amd.attn import KV8_H, Kernels, Kv8, Ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = C.create_string_buffer(4096)
AT = (C.addressof(BUF) + 15) // 16 * 16


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(library_path()):
        from nextsycl_amd.build import build
        build()
    h = C.CDLL(library_path())
    for name, (res, args) in KV8_H.items():
        f = getattr(h, name)
        f.restype, f.argtypes = res, args
    h.ns_last_error.restype = C.c_char_p
    return h


def test_the_header_and_the_table_agree():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ns_kv8.h")).read(), flags=re.S)
    assert set(KV8_H) == set(re.findall(r"\b(ns_[a-z0-9_]+)\s*\(", src))
    for name, (_, args) in KV8_H.items():
        params = re.search(name + r"\s*\((.*?)\)", src, re.S)[1]
        kinds = [C.c_void_p if "*" in a else {"int": C.c_int, "int64_t": C.c_int64, "float": C.c_float}[a.split()[0]] for a in params.split(",")]
        assert args == kinds, name


POOL = dict(Hkv=2, D=128, block=16, blocks=4, kc=AT, vc=AT, ksc=AT, vsc=AT)
STORE = dict(g=None, form=0, qt=0, k=AT, ks=256, v=AT, vs=256, T=3, start=None, lens=AT, S=3, most=1, table=AT, tmax=2, **POOL)
ATTEND = dict(g=None, form=0, qt=0, q=AT, qs=512, T=3, start=None, lens=AT, S=3, most=1, longest=100, table=AT, tmax=2, Hq=4, **POOL, win=0, scale=0.0, out=AT, acc0=None,
              acc1=None, scratch=None)
PROMPT = dict(g=None, form=0, qt=0, q=AT, qs=512, T=3, table=AT, tmax=2, p0=0, Hq=4, **POOL, win=0, scale=0.0, out=AT)
WEIGHTS = dict(g=None, form=0, qt=0, q=AT, qs=512, T=3, table=AT, tmax=2, p0=0, Hq=4, Hkv=2, D=128, block=16, blocks=4, kc=AT, ksc=AT, win=0, scale=0.0, acc0=None, acc1=AT)
EVICT = dict(g=None, form=0, lens=AT, lens1=AT, S=3, longest=100, keep=10, first=1, last=2, table=AT, to=None, tmax=2, **POOL, acc=AT)
CACHE = [dict(form=2), dict(form=-1), dict(D=64), dict(D=192), dict(block=8), dict(block=48), dict(block=256), dict(Hkv=0), dict(Hkv=40000), dict(blocks=0), dict(blocks=1 << 40), dict(tmax=0),
         dict(tmax=1 << 31), dict(kc=None), dict(ksc=None), dict(table=None), dict(kc=AT + 8)]
SEQS = [dict(S=65536)]
ROWS = [dict(qt=3), dict(qt=-1)]
QUERY = [dict(Hq=3), dict(Hq=0), dict(Hq=1 << 21), dict(qs=511), dict(q=None)]


@pytest.mark.parametrize("name,good,bad", [
    ("ns_kv8_store", STORE, CACHE + SEQS + ROWS + [dict(ks=255), dict(vs=255), dict(k=None), dict(v=None), dict(lens=None), dict(vc=None), dict(vsc=None), dict(vc=AT + 4), dict(T=1 << 31)]),
    ("ns_kv8_attend", ATTEND, CACHE + SEQS + ROWS + QUERY + [dict(most=17), dict(longest=0), dict(longest=1 << 32), dict(T=1 << 31), dict(lens=None), dict(out=None), dict(vc=None), dict(vsc=None),
                                                            dict(S=65535, most=16, Hq=8192, qs=1 << 20), dict(longest=4096), dict(acc1=AT), dict(longest=4096, scratch=AT + 4)]),
    ("ns_kv8_prompt", PROMPT, CACHE + ROWS + QUERY + [dict(p0=-1), dict(p0=1 << 31), dict(T=1 << 31), dict(out=None), dict(vc=None), dict(vsc=None)]),
    ("ns_kv8_weights", WEIGHTS, CACHE + ROWS + QUERY + [dict(p0=-1), dict(p0=1 << 31), dict(T=1 << 31), dict(acc1=None)]),
    ("ns_kv8_evict", EVICT, CACHE + SEQS + [dict(keep=0), dict(first=-1), dict(last=-1), dict(first=9), dict(last=10), dict(first=11), dict(longest=0), dict(longest=1 << 31), dict(lens=None),
                                            dict(blocks=1 << 27), dict(lens1=None), dict(acc=None), dict(vc=None), dict(vsc=None)]),
])
def test_refusals(lib, name, good, bad):
    f = getattr(lib, name)
    assert f(*good.values()) == -1 and lib.ns_last_error().decode() == name + ": a null buffer"     # (only the handle is missing)
    for change in bad:
        assert f(*{**good, **change}.values()) == -1, change
        said = lib.ns_last_error().decode()
        wants_scratch = name == "ns_kv8_attend" and (change.get("longest") == 4096 or "acc1" in change)
        assert said.startswith(name + ": ") and (said != name + ": a null buffer" or None in change.values() or wants_scratch), (change, said)


@pytest.mark.parametrize("name,good", [("ns_kv8_attend", ATTEND), ("ns_kv8_prompt", PROMPT), ("ns_kv8_weights", WEIGHTS)])
def test_query_heads_a_key_head(lib, name, good):
    """Up to 4096 of them; more are refused (a pair's row is found by a 32-bit product)."""
    for G, said in ((4096, ": a null buffer"), (4097, ": query heads a multiple of the key heads, up to 4096 times")):
        assert getattr(lib, name)(*{**good, "Hq": 2 * G, "qs": 2 * G * 128}.values()) == -1
        assert lib.ns_last_error().decode() == name + said
    assert lib.ns_kv8_attend_scratch(1, 1, 4096, 1, 128, 1000, 0) > 0 and lib.ns_kv8_attend_scratch(1, 1, 4097, 1, 128, 1000, 0) == 0


@pytest.mark.parametrize("name,good,none", [("ns_kv8_store", STORE, dict(T=0)), ("ns_kv8_store", STORE, dict(S=0)), ("ns_kv8_attend", ATTEND, dict(T=0)), ("ns_kv8_attend", ATTEND, dict(most=0)),
                                            ("ns_kv8_prompt", PROMPT, dict(T=0)), ("ns_kv8_weights", WEIGHTS, dict(T=0)), ("ns_kv8_evict", EVICT, dict(S=0))])
def test_nothing_to_do_is_no_call(lib, name, good, none):
    assert getattr(lib, name)(*{**good, **none}.values()) == 0


def test_scratch(lib):
    f = lib.ns_kv8_attend_scratch
    assert f(1, 1, 32, 8, 128, 100, 0) == 0                               # one split: no partials
    assert f(1, 1, 32, 8, 128, 100000, 0) > 0 and f(1, 1, 32, 8, 128, 100, 1) >= 32 * 102
    for bad in ((0, 1, 32, 8, 128, 100), (1, 17, 32, 8, 128, 100), (1, 1, 33, 8, 128, 100), (1, 1, 32, 8, 64, 100), (1, 1, 32, 8, 128, 0), (70000, 1, 32, 8, 128, 100), (1, 1, 32, 0, 128, 100), (65535, 16, 8192, 2, 128, 1 << 31)):
        assert f(*bad, 0) == 0 and f(*bad, 1) == 0, bad


# ---- the definition, apart from any kernel

def test_every_code_is_its_own_value():
    codes = np.arange(256).astype(np.uint8)
    for form in (INT8, E4M3):
        v = values(form, codes)
        fine = np.isfinite(v) & (np.abs(v) <= MOST[form])
        assert np.array_equal(values(form, encode(form, v[fine])), v[fine])
    assert np.nanmax(E4) == 448 and np.isnan(E4[[0x7F, 0xFF]]).all()


@pytest.mark.parametrize("form", [INT8, E4M3])
def test_a_scale_is_the_least_that_holds(form):
    for a in (1e-3, 0.7, 1.0, 126.9, 127.0, 127.1, 447.0, 448.0, 449.0, 5000.0):
        s = scale_of(form, np.array([a, -a / 3]))
        assert a <= s * MOST[form] and (a > s / 2 * MOST[form] or s == 2.0 ** HELD[form][0]) and np.log2(s) == round(np.log2(s))


def test_a_value_that_moves_between_scales_loses_less_than_a_step():
    """Re-rounding to coarser and coarser powers of two: never a step of the last one off."""
    x = np.linspace(-127, 127, 4001)
    codes, s = encode(INT8, x), 1.0
    for k in (1, 1, 2, 1):
        codes = encode(INT8, values(INT8, codes) / 2 ** k)
        s *= 2 ** k
        assert np.abs(values(INT8, codes) * s - x).max() < s


def test_the_reference_keeps_order_and_ties():
    c = Cache(INT8, 3, 1, 16, 128)
    acc = np.zeros((3, 1, 16), np.float32)
    acc[0, 0, 5], acc[1, 0, 2] = 2.0, 3.0
    k = c.k.copy()
    c.ks[:] = 1.0
    new = c.evict(acc, np.array([[0, 1]]), np.array([20]), 5, 1, 1)
    assert new[0] == 5 and acc[0, 0, :5].tolist() == [0, 0, 2, 3, 0]
    assert np.array_equal(c.k[0, 0, :5], np.stack([k[0, 0, 0], k[0, 0, 1], k[0, 0, 5], k[1, 0, 2], k[1, 0, 3]]))


# ---- the wrappers

class Buf:
    def __init__(self, n):
        self.ptr, self.len = 4096, n


def wrapped(rc=0):
    calls = []

    class Library:
        def symbol(self, name, restype, argtypes):
            def f(*a):
                calls.append((name, a))
                return 1000 if name == "ns_kv8_attend_scratch" else rc
            return C.CFUNCTYPE(restype, *argtypes)(f)

        def error(self):
            return "refused"

    return Ops(types.SimpleNamespace(raw=C.c_void_p(4096), handle=4096), Kernels(Library())), calls


def calls_of(ops):
    pool = 6 * 2 * 16 * 128
    cache = Kv8(INT8, 6, 2, 16, 128, Buf(pool), Buf(pool), Buf(48), Buf(48))
    acc = 6 * 2 * 16 * 4
    return [
        ("ns_kv8_store", lambda b: ops.kv8_store(cache, 1, b["k"], 300, b["v"], 260, 4, b["table"], 3, 2, 2, b["lens"], start=b["start"]),
         dict(k=(3 * 300 + 256) * 2, v=(3 * 260 + 256) * 2, table=24, lens=8, start=12)),
        ("ns_kv8_attend", lambda b: ops.kv8_attend(cache, 0, b["q"], 520, 4, b["table"], 3, 2, 2, 40, b["lens"], 4, b["out"], b["scratch"], start=b["start"], acc0=b["acc0"], acc1=b["acc1"]),
         dict(q=(3 * 520 + 512) * 4, out=4 * 512 * 4, table=24, lens=8, start=12, scratch=4000, acc0=acc, acc1=acc)),
        ("ns_kv8_prompt", lambda b: ops.kv8_prompt(cache, 2, b["q"], 520, 30, b["table"], 3, 7, 4, b["out"]), dict(q=(29 * 520 + 512) * 2, out=30 * 512 * 2, table=12)),
        ("ns_kv8_weights", lambda b: ops.kv8_weights(cache, 2, b["q"], 520, 30, b["table"], 3, 7, 4, b["acc0"], b["acc1"]), dict(q=(29 * 520 + 512) * 2, table=12, acc0=acc, acc1=acc)),
        ("ns_kv8_evict", lambda b: ops.kv8_evict(cache, b["acc"], b["table"], 3, 2, 40, b["lens"], b["lens1"], 10, to=b["to"]), dict(acc=acc, table=24, lens=8, lens1=8, to=24)),
    ]


@pytest.mark.parametrize("i", range(5))
@pytest.mark.parametrize("native", [True, False])
def test_the_wrappers_check_their_buffers_to_the_byte(i, native):
    ops, calls = wrapped()
    if native:
        pytest.importorskip("nextsycl_amd._ops_fast")
        assert ops._kv8_at
    else:
        ops._kv8_at = None
    name, call, need = calls_of(ops)[i]
    call({k: Buf(n) for k, n in need.items()})
    assert [c[0] for c in calls if not c[0].endswith("scratch")] == [name]
    for short in need:
        del calls[:]
        with pytest.raises(Error, match="bytes, needs"):
            call({k: Buf(n - (k == short)) for k, n in need.items()})
        assert not [c for c in calls if not c[0].endswith("scratch")]


@pytest.mark.parametrize("i", [0, 1])
@pytest.mark.parametrize("without", [(), ("start",), ("acc0", "acc1"), ("acc0",)])
def test_the_native_step_makes_the_general_ways_call(i, without):
    fast = pytest.importorskip("nextsycl_amd._ops_fast")
    assert fast.kv8_store and fast.kv8_attend
    took = []
    for general in (False, True):
        ops, calls = wrapped()
        if general:
            ops._kv8_at = None
        name, call, need = calls_of(ops)[i]
        at = {k: None if k in without else Buf(n) for k, n in need.items()}
        for j, b in enumerate(at.values()):
            if b:
                b.ptr = 1 << 20 | j << 12
        call(at)
        took.append(calls)
    assert took[0] == took[1] and len([c for c in took[0] if c[0] == name]) == 1


def test_a_refused_call_raises_once():
    ops, calls = wrapped(rc=-1)
    for i, (name, call, need) in enumerate(calls_of(ops)):
        del calls[:]
        with pytest.raises(Error, match=name[3:] + ": refused"):
            call({k: Buf(n) for k, n in need.items()})
        assert [c[0] for c in calls if not c[0].endswith("scratch")] == [name]


def test_a_pool_too_small_is_no_cache():
    pool = 6 * 2 * 16 * 128
    for short in range(4):
        with pytest.raises(Error, match="bytes, needs"):
            Kv8(INT8, 6, 2, 16, 128, *[Buf(n - (j == short)) for j, n in enumerate((pool, pool, 48, 48))])


def test_a_library_without_them_loads():
    class Library:
        def symbol(self, name, restype, argtypes):
            if name in KV8_H:
                raise OSError("lib.so: missing symbol " + name)
            return C.CFUNCTYPE(restype, *argtypes)(lambda *a: 0)

        def error(self):
            return ""

    ops = Ops(types.SimpleNamespace(raw=C.c_void_p(4096), handle=4096), Kernels(Library()))
    with pytest.raises(Error, match="missing symbol ns_kv8_attend_scratch"):
        ops.kv8_attend_scratch(1, 1, 1, 1, 128, 1)


def test_the_cpp_table_binds_every_entry_point(tmp_path):
    src = tmp_path / "kv8.cpp"
    src.write_text('#include "nextsycl_host.hpp"\n#include <cstdio>\nint main(int, char** a) { nextsycl::Api api(a[1]); nextsycl::Kv8Api k(api);'
                   ' std::printf("%lld", (long long) k.ns_kv8_attend_scratch(1, 1, 32, 8, 128, 100000, 0)); return k.ns_kv8_evict == nullptr; }\n')
    exe = tmp_path / "kv8"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe), "-ldl"], check=True)
    env = {k: v for k, v in os.environ.items() if k != "NEXTSYCL_LIB"}
    out = subprocess.run([str(exe), library_path()], capture_output=True, text=True, env=env)
    assert out.returncode == 0 and int(out.stdout) > 0, out
