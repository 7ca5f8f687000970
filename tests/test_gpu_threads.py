"""Several host threads on one handle: calls that hand data from launch to launch in the library's own scratch come out as they do alone."""
import threading

import numpy as np
import pytest

from layer_ref import BF16, F32, elt_dtype, to_type
from nextsycl_amd import DevBuf
from nextsycl_amd.attn import KV_BF16
from test_gpu_layer import random_q4

pytestmark = pytest.mark.gpu
CALLS = 300


class Products:
    """CALLS products of 16 rows whose operands go through the scratch, each into rows of its own."""

    def __init__(self, ops, qt, M, K, seed):
        g = ops.gpu
        raw, _ = to_type(qt, np.random.default_rng(seed).standard_normal((16, K)))
        self.ops, self.qt, self.M, self.K, self.one = ops, qt, M, K, 16 * M * raw.itemsize
        self.x, self.w, self.y = DevBuf.of(g, raw), DevBuf.of(g, random_q4(M, K, 64, seed)), DevBuf(g, CALLS * self.one)

    def call(self, i):
        self.ops.q4_product(self.qt, self.x, self.K, self.w, 64, self.y.view(i * self.one, self.one), self.M, 16, self.M, self.K)

    def out(self):
        return self.y.read(np.uint8).reshape(CALLS, -1)


class Prompts:
    """CALLS prompt passes over a bfloat16 cache, whose rows are widened into the scratch."""

    def __init__(self, ops, seed):
        g, r = ops.gpu, np.random.default_rng(seed)
        self.ops, self.T, self.Hq, self.Hkv, self.D = ops, 200, 8, 8, 128
        of = lambda *s: DevBuf.of(g, to_type(BF16, r.standard_normal(s))[0])  # noqa: E731
        self.q, self.k, self.v = of(self.T, self.Hq, self.D), of(self.Hkv, 256, self.D), of(self.Hkv, 256, self.D)
        self.one = self.T * self.Hq * self.D * 2
        self.y = DevBuf(g, CALLS * self.one)

    def call(self, i):
        self.ops.prompt(BF16, KV_BF16, self.q, self.Hq * self.D, self.k, self.v, self.T, self.Hq, self.Hkv, self.D, 256, 0, self.y.view(i * self.one, self.one))

    def out(self):
        return self.y.read(np.uint8).reshape(CALLS, -1)


@pytest.mark.parametrize("pair", ["products", "a product and a prompt", "prompts"])
def test_two_threads_share_a_handle(ops, pair):
    first, second = {"products": lambda: (Products(ops, F32, 64, 9000, 1), Products(ops, BF16, 4112, 5000, 2)),
                     "a product and a prompt": lambda: (Products(ops, F32, 64, 9000, 3), Prompts(ops, 4)), "prompts": lambda: (Prompts(ops, 5), Prompts(ops, 6))}[pair]()
    want = []
    for c in (first, second):
        c.call(0)
        ops.gpu.sync()
        want.append(c.out()[0].copy())
    start, errors = threading.Barrier(2), []

    def run(c):
        try:
            start.wait(60)
            for i in range(CALLS):
                c.call(i)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(c,)) for c in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    ops.gpu.sync()
    for c, w in zip((first, second), want):
        wrong = (c.out() != w).any(1)
        assert not wrong.any(), "%d of %d calls" % (wrong.sum(), CALLS)
