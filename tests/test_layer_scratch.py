"""ns_ssm_prompt_scratch of sizes that no call takes: 0, whatever they are - a size asked for ahead of its check must not end the process."""
import os
import subprocess
import sys

import pytest

from test_layer_host import lib  # noqa: F401
from nextsycl_amd import library_path

SIZES = [(100, 1, 1 << 38, 16, 1, 4), (100, 1 << 32, 1 << 32, 16, 1, 4), (100, 65537, 1, 16, 1, 4), (100, 1, 65537, 16, 1, 4), (100, 4, 4, 257, 1, 4), (100, 3, 4, 16, 2, 4), (100, 2, 4, 16, 4, 4),
         (100, 4, 4, 16, 1, 5), (100, 65536, 512, 16, 1, 4), (100, 65536, 65536, 16, 65536, 4), ((1 << 63) - 1, (1 << 63) - 1, (1 << 63) - 1, (1 << 63) - 1, (1 << 63) - 1, 4)]


@pytest.mark.parametrize("size", SIZES)
def test_sizes_that_no_call_takes(lib, size):  # noqa: F811
    # (in a process of its own: a division by zero ends one)
    code = "import ctypes, sys; f = ctypes.CDLL(%r).ns_ssm_prompt_scratch; f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_int64] * 6; print(f(*map(int, sys.argv[1:])))" % library_path()
    r = subprocess.run([sys.executable, "-c", code] + [str(v) for v in size], capture_output=True, text=True, timeout=120, env=dict(os.environ))
    assert r.returncode == 0 and r.stdout.strip() == "0", (r.returncode, r.stdout, r.stderr[-300:])


def test_sizes_at_the_limits(lib):  # noqa: F811
    f = lib.ns_ssm_prompt_scratch
    for T, H, P, N, G, K in ((100, 65536, 1, 1, 1, 1), (100, 1, 65536, 256, 1, 4), ((1 << 63) - 1, 1, 1, 1, 1, 4), (100, 65536, 255, 1, 1, 4)):
        assert f(T, H, P, N, G, K) > 0
