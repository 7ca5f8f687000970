"""The most that one call of the hybrid layers' norms and 4-bit products takes (include/ns_layer.h): what one launch holds, refused by name past it and
before any GPU is touched. Calls within it end at the null handle."""
import pytest

from test_layer_host import GATED, PACK, PRODUCT, RESID, lib  # noqa: F401

MOST = (1 << 32) - 1


def most_rows(n, qt):
    """By the header: fewer than 2^32 threads, 64 a unit of up to 64 pieces (in blocks of 256), else 64 for each 64 pieces, 1024 at most."""
    per = 16 // (2 if qt else 4)
    pieces = n if n % per and n <= 64 else -(-n // per)
    if pieces <= 64:
        return MOST // 256 * 4
    if pieces <= 1024:
        return MOST // (-(-pieces // 64) * 64)
    if pieces <= 2048:
        return MOST // (-(-pieces // 128) * 64)          # (two pieces a thread)
    return MOST // 1024


@pytest.mark.parametrize("qt", [0, 1, 2])
@pytest.mark.parametrize("n", [1, 35, 64, 65, 256, 257, 512, 513, 520, 4096, 4100, 8200, 16384, 16400, 40000])
def test_rows_of_the_norms(lib, qt, n):  # noqa: F811
    most = most_rows(n, qt)
    for name, good, groups in (("ns_norm_gated", GATED, 2), ("ns_norm_gated", GATED, 1), ("ns_norm_residual", RESID, 1)):
        D, f = n * groups, getattr(lib, name)
        size = dict(D=D, qt=qt, **(dict(groups=groups, ys=D, zs=D, os=D) if name == "ns_norm_gated" else dict(xs=D, hs=D, h1s=D, os=D)))
        for T, said in ((most // groups, "a null buffer"), (most // groups + 1, "too many rows"), ((1 << 63) - 1, "too many rows")):
            assert f(*{**good, **size, "T": T}.values()) == -1 and lib.ns_last_error().decode() == name + ": " + said, T


def test_4_bit_weights(lib):  # noqa: F811
    f = lib.ns_q4_product
    for M, said in (((1 << 27) - 16, "a null buffer"), ((1 << 27) - 15, "up to 2^27 - 16 outputs, 1 to 2^22 inputs")):
        assert f(*{**PRODUCT, "M": M, "ys": M}.values()) == -1 and lib.ns_last_error().decode() == "ns_q4_product: " + said
    f = lib.ns_q4_pack
    for M, K, group, said in (((1 << 26) - 16, 128 * 16, 32, "a null buffer"), (1 << 26, 128 * 16, 32, "too many weights"), (1 << 26, 128 * 16, 64, "a null buffer"),
                              (1 << 30, 1 << 30, 128, "too many weights")):
        assert f(*{**PACK, "M": M, "K": K, "ss": K, "group": group}.values()) == -1 and lib.ns_last_error().decode() == "ns_q4_pack: " + said, (M, K, group)
