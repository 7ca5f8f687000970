"""The built code of the hybrid layers' kernels (include/ns_layer.h): no vector register of theirs is spilled - the scans were two to three
times as slow where some were."""
import re

import pytest

from test_code_objects import _over_code_objects


@pytest.fixture(scope="module")
def spilled():
    """{kernel: vector registers spilled}"""
    kernels = [k for text in _over_code_objects("llvm-readelf", "--notes") for k in text.split("\n  - .agpr_count:")[1:]]
    return {re.search(r"^    \.name: +(\S+)$", k, re.M)[1]: int(re.search(r"\.vgpr_spill_count: +(\d+)", k)[1]) for k in kernels}


@pytest.mark.parametrize("kernel,least", [("ssm_prep_kernel", 9), ("ssm_scan_kernel", 54), ("ssm_step_kernel", 30), ("norm_gated_kernel", 30), ("norm_residual_kernel", 50),
                                          ("q4_product_kernel", 36), ("q4_rows_kernel", 3), ("q4_pack_kernel", 1)])
def test_no_vector_registers_are_spilled(spilled, kernel, least):
    found = {n: c for n, c in spilled.items() if kernel in n}
    assert len(found) >= least, found
    assert not any(found.values()), found
