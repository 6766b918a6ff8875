"""Sizes past what a launch can have (2^32 threads) are refused with the sizes that were given, and not by the runtime."""
import pytest

from gaac_amd import _lib

A = 16      # an address that nothing reads


@pytest.mark.parametrize("name,args", [
    ("gaac_fp4_append", [A, 1 << 24, 2, 4, A, A, 512, 128, 512, 128, A, 2, 64, A, A, None]),
    ("gaac_fp4_attn", [A, A, A, 2, 2, 64, A, 1 << 20, 8, 8, 1.0, 1, A, A, A, None]),
    ("gaac_fp4_attn", [A, A, A, 2, 2, 64, A, 1 << 10, 8, 8, 1.0, 1 << 10, A, A, A, None]),
    ("gaac_qk_norm_rope", [0, A, A, 512, 128, 512, 128, 1 << 26, 4, 4, 128, 128, None, None, 0, 0, 1e-6, A, 0, A, A, 10, 0, A, A, None]),
])
def test_refused_by_name(name, args):
    with pytest.raises(RuntimeError, match=f"{name} failed .-1.: {name}: bad sizes"): _lib.call(name, *args)
