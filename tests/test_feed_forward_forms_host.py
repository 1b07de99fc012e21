"""Which form each product of the feed-forward operators takes, asked of the library without a device: the cases of
test_gpu_feed_forward_tiles.py are of every form, kind and type that there is."""
import ctypes

import test_gpu_feed_forward_tiles as tiles


def test_every_form_has_a_case():
    each = list(tiles.cases())
    for product, form, dtype, m, n, k in each:
        assert tiles.form_of(product, dtype, m, n, k) == form, (product, form, dtype, m, n, k)
    found = {(c[0], c[1], c[2]) for c in each}
    tile_forms = (tiles.LARGE, tiles.TALL, tiles.MIDDLE, tiles.SMALL)
    for dtype in tiles.CODE:
        for form in range(8):
            assert (tiles.LINEAR, form, dtype) in found
            assert ((tiles.GATED, form, dtype) in found) == (form != tiles.ROWS_64 or dtype == tiles.F32)
        if dtype == tiles.E4M3:
            continue
        for form in tile_forms:
            for product in (tiles.LINEAR_DZ, tiles.GATED_DZ, tiles.LINEAR_DW, tiles.GATED_DW):
                assert (product, form, dtype) in found
        for form in (*tile_forms, tiles.SMALL_BY_FOUR):
            assert (tiles.LINEAR_DX, form, dtype) in found and (tiles.GATED_DX, form, dtype) in found


def test_no_other_form_is_taken():
    """Over sizes of all kinds: dz and dW never share a contraction in a workgroup, a gated result of 16 or 8 bits never takes 64 rows."""
    for dtype in tiles.CODE:
        for product in range(2 if dtype == tiles.E4M3 else 8):
            for m in (1, 16, 17, 33, 45, 48, 64, 100, 400, 1100, 4090, 9000):
                for n in (1, 40, 300, 1101, 1360, 1361, 2101, 4100, 9000):
                    for k in (1, 100, 1500, 5000):
                        form = tiles.form_of(product, dtype, m, n, k)
                        if product >= tiles.LINEAR_DZ:
                            assert form <= tiles.SMALL_BY_FOUR
                            assert form < tiles.SMALL_BY_FOUR or product in (tiles.LINEAR_DX, tiles.GATED_DX)
                        if product == tiles.GATED and dtype != tiles.F32:
                            assert form != tiles.ROWS_64


def test_form_refusals():
    from verace_amd import _lib
    call, form = _lib.load().vmi_feed_forward_form, ctypes.c_int(-1)
    INVALID = 1
    assert call(0, 1, 0, 8, 8, 8, ctypes.byref(form)) == 0 and form.value == tiles.ROWS_16
    for args in ((8, 1, 1, 8, 8, 8), (-1, 1, 1, 8, 8, 8), (0, 4, 0, 8, 8, 8), (0, 1, 3, 8, 8, 8), (1, 1, 0, 8, 8, 8), (2, 3, 1, 8, 8, 8),
                 (0, 1, 0, -1, 8, 8), (0, 1, 0, 8, (1 << 30) + 1, 8)):
        assert call(*args, ctypes.byref(form)) == INVALID, args
    assert call(0, 1, 0, 8, 8, 8, None) == INVALID
