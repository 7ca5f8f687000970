"""What a prompt writes into its scratch."""
import numpy as np
import pytest

from layer_ref import BF16, F16, F32, Layer
from test_gpu_ssm_edges import Call, rows_of

pytestmark = pytest.mark.gpu


def test_bfloat16_rows_leave_out_what_their_scan_does_not_read(ops):
    """C's operands are two halfs a value for float32 and half rows; the scan of bfloat16 rows takes the first: the others' 64 x 128 x 2 bytes a chunk are
    neither made nor written."""
    L, T = Layer(2, 64, 128, 1, 4, seed=1), 128
    left = {}
    for qt in (F32, F16, BF16):
        c = Call(ops, L, qt, rows_of(L, qt, T, 2)[0])
        c.sc.fill(0xAB)
        c.run()
        ops.gpu.sync()
        left[qt] = int((c.sc.read(np.uint32) == 0xABABABAB).sum()) * 4
    assert left[F32] == left[F16] and left[BF16] - left[F32] == T * 128 * 2, left
