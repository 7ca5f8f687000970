"""The built code of the kernels over 8-bit caches in blocks (include/ns_kv8.h): no vector register of theirs is spilled - a register's way back from memory
would wait for the transfers that their counted waits leave in flight."""
import re

import pytest

from test_code_objects import _over_code_objects


@pytest.fixture(scope="module")
def spilled():
    """{kernel: vector registers spilled}"""
    kernels = [k for text in _over_code_objects("llvm-readelf", "--notes") for k in text.split("\n  - .agpr_count:")[1:]]
    return {re.search(r"^    \.name: +(\S+)$", k, re.M)[1]: int(re.search(r"\.vgpr_spill_count: +(\d+)", k)[1]) for k in kernels}


@pytest.mark.parametrize("kernel,count", [("kv8_store_kernel", 48), ("kv8_widen_kernel", 4), ("kv8_attend_kernel", 36), ("kv8_join_kernel", 12),
                                          ("kv8_rows_kernel", 6), ("kv8_pass_kernel", 16), ("kv8_stats_join_kernel", 1), ("kv8_columns_join_kernel", 1),
                                          ("kv8_select_kernel", 3), ("kv8_move_kernel", 8), ("kv8_settle_kernel", 1)])
def test_no_vector_registers_are_spilled(spilled, kernel, count):
    found = {n: c for n, c in spilled.items() if kernel in n}
    assert len(found) == count and not any(found.values()), found
