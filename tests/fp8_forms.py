"""Sizes at which every form of the products of rows in 8 bits is taken, with every number of blocks of K that can be left over at its end.

{outputs in 32 bits, gated: {form: (M, N, numbers of blocks)}}; K is 5 less than the blocks hold, M and N end inside a tile.  A gated pair has no form 0 (one tile of weights a block)."""
import ctypes

from gaac_amd import _lib

FEW, MANY, TWELVE = (33, 34, 35, 36), (5, 6, 7, 8), tuple(range(13, 25))      # eight waves that share K out by fours, and each comes round again | steps by fours | by twelves
SIZES = {
    (False, False): {0: (5, 67, FEW), 1: (13, 4101, FEW), 2: (1361, 33, FEW), 3: (4101, 33, FEW), 4: (2593, 65, MANY), 5: (65, 8231, MANY), 6: (193, 16439, MANY), 7: (259, 8389, MANY), 8: (965, 10897, MANY),
                     9: (257, 10913, TWELVE)},
    (False, True): {1: (5, 67, FEW), 2: (33, 17, FEW), 3: (4141, 17, FEW), 4: (65, 1305, MANY), 5: (65, 4101, MANY), 6: (193, 8241, MANY), 7: (257, 4109, MANY), 8: (385, 11013, MANY), 9: (257, 5517, TWELVE)},
    (True, False): {0: (5, 67, FEW), 1: (13, 4113, FEW), 2: (65, 1653, FEW), 3: (1365, 33, FEW), 4: (65, 4103, MANY), 5: (129, 10883, MANY)},
    (True, True): {1: (5, 67, FEW), 2: (65, 817, FEW), 3: (65, 17, FEW), 4: (65, 2051, MANY), 5: (129, 5519, MANY)},
}
CASES = [(wide, gated, form, M, N, 128 * blocks - 5) for (wide, gated), forms in SIZES.items() for form, (M, N, all_blocks) in forms.items() for blocks in all_blocks]


def form_of(M: int, N: int, K: int, gated: bool, wide: bool) -> int:
    """The form that the library takes for these sizes; wide: outputs in 32 bits."""
    form = ctypes.c_int(-1)
    _lib.call("gaac_fp8_product_form", M, N, K, int(gated), 2 if wide else 0, ctypes.addressof(form))
    return form.value
