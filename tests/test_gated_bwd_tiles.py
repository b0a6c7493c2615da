"""How gated_linear's backward products are cut: the sizes of the GPU tests reach every
width of a block, with its contraction whole and in parts (no GPU needed)."""
import ctypes as C

import pytest

from neutrongt_amd import _lib

# (rows, n_out, n_in): columns of a block and whether the contraction is cut, of dx and of
# dW; rows, outputs and widths that are whole tiles, whole pieces and neither
SIZES = {
    (32862, 8, 132): ((192, False), (128, True)),
    (33000, 72, 392): ((192, False), (128, True)),
    (65536, 16, 192): ((192, False), (192, True)),
    (8, 27755, 146): ((192, True), (192, False)),
    (9, 28160, 152): ((192, True), (192, False)),
    (65, 33001, 192): ((128, True), (192, False)),
    (70, 17000, 769): ((128, True), (192, False)),
    (54211, 9, 132): ((192, False), (192, True)),
    (66000, 8, 192): ((192, False), (192, True)),
    (36518, 8, 194): ((256, False), (128, True)),
    (66000, 72, 200): ((256, False), (128, True)),
    (33001, 64, 761): ((256, False), (128, True)),
    (8, 37455, 195): ((256, True), (256, False)),
    (9, 38016, 256): ((256, True), (256, False)),
    (65, 33001, 250): ((128, True), (256, False)),
    (65, 16500, 768): ((128, True), (256, False)),
    (97080, 8, 194): ((256, False), (256, True)),
    (98304, 8, 256): ((256, False), (256, True)),
    (40, 60, 136): ((128, False), (128, False)),
    (5000, 2100, 1000): ((192, True), (256, True)),
}


def _tiles(size, rc=0):
    columns, splits = (C.c_int32 * 2)(), (C.c_int32 * 2)()
    assert _lib.load().ngt_gated_bwd_tiles(*size, columns, splits) == rc
    return tuple((c, s > 1) for c, s in zip(columns, splits))


@pytest.mark.parametrize("size", list(SIZES))
def test_the_cut_of_a_size(size):
    assert _tiles(size) == SIZES[size]


def test_every_cut_is_among_them():
    for product in (0, 1):
        assert {cut[product] for cut in SIZES.values()} == {(c, s) for c in (128, 192, 256)
                                                            for s in (False, True)}


def test_refusals():
    lib, two = _lib.load(), (C.c_int32 * 2)()
    for size, code in (((-1, 8, 8), 1), ((4, 0, 8), 1), ((4, 8, 0), 1), ((4, 1 << 20, 8), 2)):
        _tiles(size, code)
    assert lib.ngt_gated_bwd_tiles(4, 8, 8, None, two) == 1
    assert lib.ngt_gated_bwd_tiles(4, 8, 8, two, None) == 1
    assert _tiles((0, 8, 8)) == ((256, False), (256, False))  # nothing is launched
