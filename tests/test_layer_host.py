"""What the hybrid layers' entry points (include/ns_layer.h) refuse, through the C ABI and before any GPU is touched, and
their sizes. Arguments that nothing is wrong with end at the null handle."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

from layer_ref import q4_weights
from nextsycl_amd import library_path
from nextsycl_amd.attn import LAYER_H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = C.create_string_buffer(4096)
AT = (C.addressof(BUF) + 15) // 16 * 16


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(library_path()):
        from nextsycl_amd.build import build
        build()
    h = C.CDLL(library_path())
    for name, (res, args) in LAYER_H.items():
        f = getattr(h, name)
        f.restype, f.argtypes = res, args
    h.ns_last_error.restype = C.c_char_p
    return h


def test_the_header_and_the_table_agree(lib):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ns_layer.h")).read(), flags=re.S)
    assert set(LAYER_H) == set(re.findall(r"\b(ns_[a-z0-9_]+)\s*\(", src))


PROMPT = dict(g=None, qt=0, xbc=AT, xs=100, dt=AT, dts=2, cw=AT, cb=None, a=AT, dtb=None, d=None, lo=0.0, hi=float("inf"), conv=AT, cap=4, p0=0, T=3, H=2, P=4,
              N=8, G=1, K=4, h0=None, h1=AT, y=AT, ys=8, scratch=AT)
STEP = dict(g=None, qt=0, xbc=AT, xs=100, dt=AT, dts=2, cw=AT, cb=None, a=AT, dtb=None, d=None, lo=0.0, hi=float("inf"), conv=AT, cap=4, p0=0, pos=None, slots=None,
            nslots=3, R=3, H=2, P=4, N=8, G=1, K=4, h0=None, h1=AT, y=AT, ys=8)
GATED = dict(g=None, qt=0, y=AT, ys=16, z=AT, zs=16, w=None, out=AT, os=16, T=1, D=16, groups=2, eps=1e-5, order=0)
RESID = dict(g=None, qt=1, rt=0, x=AT, xs=16, h=AT, hs=16, h1=AT, h1s=16, out=AT, os=16, T=1, D=16, eps=1e-5, scale=1.0, post=None, gate=None, pre=None)
PACK = dict(g=None, form=0, src=AT, ss=64, M=4, K=64, group=32, w=AT)
PRODUCT = dict(g=None, qt=0, x=AT, xs=64, w=AT, group=32, y=AT, ys=4, T=2, M=4, K=64)
ONE = [dict(qt=3), dict(qt=-1), dict(H=0), dict(P=0), dict(N=0), dict(G=0), dict(N=257), dict(H=3, G=2, xs=1000), dict(K=0), dict(K=5), dict(xs=23), dict(dts=1), dict(ys=7), dict(lo=2.0, hi=1.0),
       dict(lo=float("nan")), dict(p0=-1), dict(H=1 << 40), dict(P=1 << 40), dict(xbc=None), dict(dt=None), dict(cw=None), dict(a=None), dict(h1=None), dict(y=None), dict(conv=None)]


@pytest.mark.parametrize("name,good,bad", [
    ("ns_ssm_prompt", PROMPT, ONE + [dict(cap=2), dict(cap=0), dict(scratch=None)]),
    ("ns_ssm_step", STEP, ONE + [dict(cap=3), dict(R=4), dict(R=4097, nslots=5000), dict(nslots=0), dict(nslots=1 << 40)]),
    ("ns_norm_gated", GATED, [dict(qt=3), dict(groups=0), dict(groups=3), dict(order=2), dict(ys=15), dict(zs=15), dict(os=15), dict(y=None), dict(z=None), dict(out=None), dict(D=1 << 25, groups=1)]),
    ("ns_norm_residual", RESID, [dict(qt=3), dict(rt=2), dict(rt=-1), dict(xs=15), dict(hs=15), dict(h1s=15), dict(os=15), dict(h=None), dict(h1=None, out=None), dict(x=None, post=AT),
                                 dict(x=None, gate=AT), dict(D=1 << 25)]),
    ("ns_q4_pack", PACK, [dict(form=2), dict(group=16), dict(group=256), dict(form=1, group=64), dict(form=1, K=40), dict(ss=63), dict(src=None), dict(w=None), dict(w=AT + 4), dict(K=1 << 31, ss=1 << 31)]),
    ("ns_q4_product", PRODUCT, [dict(qt=5), dict(T=17), dict(group=48), dict(K=0), dict(xs=63), dict(ys=3), dict(x=None), dict(w=None), dict(y=None), dict(w=AT + 8)]),
])
def test_refusals(lib, name, good, bad):
    f = getattr(lib, name)
    assert f(*good.values()) == -1 and lib.ns_last_error().decode() == name + ": a null buffer"     # (only the handle is missing)
    for change in bad:
        assert f(*{**good, **change}.values()) == -1, change
        said = lib.ns_last_error().decode()
        assert said.startswith(name + ": ") and (said != name + ": a null buffer" or None in change.values()), (change, said)


@pytest.mark.parametrize("name,good,none", [("ns_ssm_prompt", PROMPT, dict(T=0)), ("ns_ssm_step", STEP, dict(R=0)), ("ns_norm_gated", GATED, dict(T=0)), ("ns_norm_residual", RESID, dict(D=0)),
                                            ("ns_q4_pack", PACK, dict(M=0)), ("ns_q4_product", PRODUCT, dict(T=0))])
def test_nothing_to_do_is_no_call(lib, name, good, none):
    assert getattr(lib, name)(*{**good, **none}.values()) == 0


def test_sizes(lib):
    assert lib.ns_q4_bytes(16, 128, 32) == 1152 and lib.ns_q4_bytes(17, 129, 128) == 4 * 1056 and lib.ns_q4_bytes(1, 1, 64) == 1088
    assert lib.ns_q4_bytes(0, 5, 32) == 0 and lib.ns_q4_bytes(5, 5, 33) == 0
    f = lib.ns_ssm_prompt_scratch
    assert f(0, 8, 64, 128, 1, 4) == 0 and f(1, 8, 64, 128, 1, 4) > 0
    # bounded, however long the prompt
    assert f(1 << 20, 8, 64, 128, 1, 4) == f(8192, 8, 64, 128, 1, 4)


def test_the_layout_of_4_bit_weights_is_a_permutation():
    """Every nibble and every scale of a tile is some (row, value)'s."""
    for group in (32, 64, 128):
        gr = 128 // group
        m, k = np.arange(16)[:, None], np.arange(128)[None]
        e = k % 8
        nib = 2 * (16 * (m + 16 * (k // 8 % 4)) + 4 * (k // 32) + (e % 2) * 2 + e // 4) + (e // 2) % 2
        assert np.array_equal(np.sort(nib.ravel()), np.arange(2048))
        sc = m // 4 * 4 * gr + k // group * 4 + m % 4
        assert np.array_equal(np.unique(sc), np.arange(16 * gr)) and (np.bincount(sc.ravel()) == group).all()
    w = np.zeros((1, 1, 1056), np.uint8)
    w[:, :, 1024:] = np.ones(16, np.float16).view(np.uint8)
    w[0, 0, 16 * (3 + 16 * 1) + 4 * 2 + 2 + 0] = 0xF0             # row 3, value 64 + 8 + 3: byte 2, the high nibble
    _, q, _ = q4_weights(w, 16, 128, 128)
    assert q[3, 64 + 8 + 3] == 15 and q.sum() == 15


# ---- the wrappers' native step (csrc/ops_fast.c): the call the general way makes, or none

class Buf:
    def __init__(self, ptr, n):
        self.ptr, self.len = ptr, n


def recorded(rc=0):
    """An Ops over entry points that note their arguments, and the notes."""
    import types

    from nextsycl_amd.attn import Ops
    notes, keep = [], []

    def entry(name):
        res, args = LAYER_H[name]

        def f(*a):
            if name == "ns_q4_bytes":
                return 5000
            notes.append((name, a))
            return rc
        keep.append(C.CFUNCTYPE(res, *args)(f))
        return keep[-1]

    k = types.SimpleNamespace(keep=keep, api=types.SimpleNamespace(error=lambda: "refused"), **{n[3:]: entry(n) for n in LAYER_H})
    return Ops(types.SimpleNamespace(raw=C.c_void_p(4096), handle=4096), k), notes


def layer_calls(qt):
    """name -> (arguments by name, the buffers' least sizes, the buffers that may be None)."""
    e, T, D, H, P, N, G, K, cap, slots = {0: 4, 1: 2, 2: 2}[qt], 3, 48, 4, 8, 6, 2, 4, 7, 5
    chan = H * P + 2 * G * N
    rows = lambda stride, last, e=e: ((T - 1) * stride + last) * e  # noqa: E731
    return {
        "norm_gated": (dict(qt=qt, ys=50, zs=52, os=49, T=T, D=D, groups=2, eps=1e-5, order=1), dict(y=rows(50, D), z=rows(52, D), out=rows(49, D), w=4 * D), ["w"]),
        "norm_residual": (dict(qt=qt, rt=0, xs=50, hs=52, h1s=49, os=51, T=T, D=D, eps=1e-5, scale=0.5),
                          dict(x=rows(50, D), h=rows(52, D, 4), h1=rows(49, D, 4), out=rows(51, D), post=4 * D, gate=4 * D, pre=4 * D), ["x", "h1", "out", "post", "gate", "pre"]),
        "q4_product": (dict(qt=qt, xs=70, group=64, ys=40, T=T, M=33, K=65), dict(x=rows(70, 65), w=5000, y=rows(40, 33)), []),
        "ssm_step": (dict(qt=qt, xs=chan + 9, dts=chan + 9, cap=cap, p0=11, R=T, H=H, P=P, N=N, G=G, K=K, ys=H * P + 2, nslots=slots, dt_lo=0.01, dt_hi=float("inf")),
                     dict(xbc=rows(chan + 9, chan), dt=rows(chan + 9, H), cw=chan * K * 4, cb=chan * 4, a=H * 4, dtb=H * 4, d=H * 4, conv=slots * cap * chan * 4,
                          h0=slots * H * P * N * 4, h1=slots * H * P * N * 4, y=rows(H * P + 2, H * P), slots=T * 4, pos=T * 4), ["cb", "dtb", "d", "h0", "slots", "pos"]),
    }


@pytest.mark.parametrize("name", ["norm_gated", "norm_residual", "q4_product", "ssm_step"])
@pytest.mark.parametrize("qt", [0, 1, 2])
def test_the_native_step_makes_the_general_ways_call(name, qt):
    from nextsycl_amd import Error
    fast = pytest.importorskip("nextsycl_amd._ops_fast")
    args, need, optional = layer_calls(qt)[name]
    bufs = {b: Buf(1 << 20 | i << 12, n) for i, (b, n) in enumerate(need.items())}
    for without in [None] + optional:
        given = dict(bufs, **({without: None} if without else {}))
        got, took = [], []
        for general in (False, True):
            ops, notes = recorded()
            native = getattr(fast, name)
            if general:
                ops._layer_at = None
            else:
                assert ops._layer_at
            getattr(ops, name)(**args, **given)
            took.append(native)
            assert len(notes) == 1
            got.append(notes[0])
        assert got[0] == got[1], without
    for b in need:
        short, words = dict(bufs), []
        short[b] = Buf(bufs[b].ptr, need[b] - 1)
        for general in (False, True):
            ops, notes = recorded()
            if general:
                ops._layer_at = None
            with pytest.raises(Error) as err:
                getattr(ops, name)(**args, **short)
            words.append(str(err.value))
            assert not notes
        assert words[0] == words[1]
    # a failure is raised once, behind one call; an entry replaced on the kernels is the one that is called
    ops, notes = recorded(rc=-1)
    with pytest.raises(Error, match="refused"):
        getattr(ops, name)(**args, **bufs)
    assert len(notes) == 1
    ops, notes = recorded()
    other = []
    setattr(ops.k, name, lambda *a: other.append(a) or 0)
    getattr(ops, name)(**args, **bufs)
    assert len(other) == 1 and not notes


@pytest.mark.parametrize("name,good", [("ns_ssm_prompt", PROMPT), ("ns_ssm_step", STEP)])
def test_positions_past_any_sequence(lib, name, good):
    f = getattr(lib, name)
    assert f(*{**good, "p0": (1 << 62) + 1}.values()) == -1 and "positions" in lib.ns_last_error().decode()
    assert f(*{**good, "p0": (1 << 62) - 1}.values()) == -1 and lib.ns_last_error().decode() == name + ": a null buffer"


def test_rows_too_far_apart_and_scratch_off_its_alignment(lib):
    g = C.create_string_buffer(1 << 16)        # (a handle that is not looked at: the call ends in front of any use of it)
    for change, word in ((dict(xs=(1 << 23) + 1), "apart"), (dict(scratch=AT + 4), "aligned")):
        assert lib.ns_ssm_prompt(*{**PROMPT, "g": C.addressof(g), **change}.values()) == -1
        assert word in lib.ns_last_error().decode()


def test_a_cpp_host_binds_the_layers(lib, tmp_path):
    """LayerApi of include/nextsycl_host.hpp: every entry point of the header, called through the table."""
    src, exe = tmp_path / "layers.cpp", tmp_path / "layers"
    src.write_text("""#include <cstdio>
#include "nextsycl_host.hpp"
int main() {
    const nextsycl::Api api;
    const nextsycl::LayerApi layers(api);
    int bound = 0;
#define COUNT(name) bound += layers.name != nullptr;
    NS_HOST_LAYER_SYMBOLS(COUNT)
    const int rc = layers.ns_norm_gated(nullptr, 3, nullptr, 1, nullptr, 1, nullptr, nullptr, 1, 1, 1, 1, 0.0f, 0);
    std::printf("%d %lld %lld %d %s\\n", bound, (long long) layers.ns_q4_bytes(17, 129, 128), (long long) layers.ns_ssm_prompt_scratch(0, 1, 1, 1, 1, 1), rc,
                api.error().c_str());
}
""")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe), "-ldl"], check=True)
    out = subprocess.run([str(exe)], env=dict(os.environ, NEXTSYCL_LIB=library_path()), check=True, capture_output=True, text=True, timeout=120).stdout
    assert out.startswith("%d %d 0 -1 ns_norm_gated: " % (len(LAYER_H), 4 * 1056)), out
