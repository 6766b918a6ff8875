"""The rule by which a product takes its form, without a GPU: the sizes of the forms' tests reach all of them."""
import random

import pytest

from fp8_forms import CASES, SIZES, form_of
from gaac_amd import _lib


@pytest.mark.parametrize("wide,gated", SIZES)
def test_every_case_takes_its_form(wide, gated):
    for w, g, form, M, N, K in CASES:
        if (w, g) == (wide, gated): assert form_of(M, N, K, g, w) == form, (M, N, K)


@pytest.mark.parametrize("wide,gated", SIZES)
def test_no_size_takes_a_form_that_has_no_case(wide, gated):
    rng = random.Random(1)
    log = lambda a, b: round(a * (b / a) ** rng.random())
    seen = {form_of(log(1, 1 << 20), log(1, 1 << 22), log(1, 65536), gated, wide) for _ in range(20000)} | {form_of(log(1, 8192), log(16, 32768), log(128, 16384), gated, wide) for _ in range(20000)}
    assert seen == set(SIZES[wide, gated])


def test_refusals():
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), ((1 << 20) + 1, 1, 1), (1, (1 << 22) + 1, 1), (1, 1, 65537)):
        with pytest.raises(RuntimeError, match="gaac_fp8_product_form failed .*bad sizes"): form_of(*bad, False, False)
    with pytest.raises(RuntimeError, match="null pointer"): _lib.call("gaac_fp8_product_form", 1, 1, 1, 0, 0, None)
    with pytest.raises(RuntimeError, match="type must be"): _lib.call("gaac_fp8_product_form", 1, 1, 1, 0, 3, 16)
