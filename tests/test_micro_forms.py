"""Each kernel of the microscaled products and of the experts', at sizes that it takes: the calls' own rules say which, so that
a rule set to other figures cannot leave a kernel without a test."""
import ctypes

import pytest

import test_gpu_experts as experts_base
import test_gpu_micro as base

TYPES = {"f32": 0, "bf16": 1, "f16": 2}
FORMATS = {"e4m3": 0, "e2m1": 1}


def product_form(rows, inner, outer, dtype, codes, call="linear"):
    from tcc_spmm_amd._lib import check, lib
    form = ctypes.c_char_p()
    check(getattr(lib(), f"tcc_{call}_micro_form")(rows, inner, outer, TYPES[dtype], FORMATS[codes], ctypes.byref(form)))
    return form.value.decode()


def expert_form(choices, count, inner, outer, dtype, codes):
    from tcc_spmm_amd._lib import check, lib
    form = ctypes.c_char_p()
    check(lib().tcc_matmul_experts_form(choices, count, inner, outer, TYPES[dtype], FORMATS[codes], ctypes.byref(form)))
    return form.value.decode()


EIGHT, FOUR, EXACT = (("bf16", "e4m3"), ("f16", "e4m3")), tuple((t, "e2m1") for t in TYPES), (("f32", "e4m3"),)
# Odd and even numbers of steps and of dwords of exponents, ragged edges, one tile and many.
PRODUCTS = [
    *(("microWide", *kind, *size) for kind in EIGHT for size in ((3900, 600, 4000), (3000, 2000, 3000), (4000, 900, 4090))),
    *(("microWide", *kind, *size) for kind in FOUR for size in ((3900, 600, 4000), (4097, 1153, 4000), (3000, 2000, 3000))),
    *(("microTiles128", *kind, 4091, 300, 4099) for kind in EIGHT + FOUR),
    *(("microTiles64", *kind, *size) for kind in EIGHT + FOUR + EXACT for size in ((777, 1001, 1437), (1900, 1500, 2300))),
    *(("microTiles64x32", *kind, *size) for kind in EIGHT + FOUR + EXACT for size in ((48, 4096, 8191), (500, 2900, 1001), (192, 4100, 2500))),
    *(("microTiles32", *kind, *size) for kind in EIGHT + FOUR + EXACT for size in ((16, 4096, 1000), (32, 2900, 513), (17, 130, 40))),
    *(("microTokens", *kind, *size) for kind in EIGHT + FOUR + EXACT for size in ((1, 4096, 130), (3, 100, 77), (7, 4096, 300), (16, 1001, 50))),
]

# tokens, each, experts, inner, outer
EXPERTS = [
    *(("microWide", *kind, *size) for kind in EIGHT + FOUR for size in ((3001, 2, 8, 1000, 2048), (6000, 2, 4, 1200, 900))),
    ("microWide", "bf16", "e2m1", 15000, 2, 70, 1000, 520),  # more experts than a wave has lanes, several tiles a workgroup
    *(("microTiles128", *kind, 3001, 2, 8, 2048, 1000) for kind in EIGHT + FOUR),
    ("microTiles128", "f16", "e4m3", 15000, 2, 70, 1000, 520),
    *(("microTiles64", *kind, *size) for kind in EIGHT + FOUR + EXACT for size in ((24, 4, 32, 2048, 400), (400, 2, 8, 300, 129),
                                                                                 (90, 3, 200, 130, 70))),
]


def test_the_sizes_below_take_every_kernel():
    for form, dtype, codes, rows, inner, outer in PRODUCTS:
        assert product_form(rows, inner, outer, dtype, codes) == form, (dtype, codes, rows, inner, outer)
        given = product_form(rows, inner, outer, dtype, codes, "matmul")
        assert given == form or form == "microTokens" and given != form
    for form, dtype, codes, tokens, each, count, inner, outer in EXPERTS:
        assert expert_form(tokens * each, count, inner, outer, dtype, codes) == form, (dtype, codes, tokens, inner, outer)
    # each pair of types that a kernel is built for
    built = {("microWide", *k) for k in EIGHT + FOUR} | {("microTiles128", *k) for k in EIGHT + FOUR} | {
        (name, *k) for name in ("microTiles64", "microTiles64x32", "microTiles32", "microTokens") for k in EIGHT + FOUR + EXACT}
    assert {p[:3] for p in PRODUCTS} == built
    assert {p[:3] for p in EXPERTS} == {b for b in built if b[0] not in ("microTiles64x32", "microTiles32", "microTokens")}


@pytest.mark.gpu
@pytest.mark.parametrize("form,dtype,codes,rows,inner,outer", PRODUCTS)
def test_products(gpu, form, dtype, codes, rows, inner, outer):
    base.test_linear(gpu, rows, inner, outer, dtype, codes)


@pytest.mark.gpu
@pytest.mark.parametrize("form,dtype,codes,tokens,each,count,inner,outer", EXPERTS)
def test_experts(gpu, form, dtype, codes, tokens, each, count, inner, outer):
    experts_base.test_linear_experts(gpu, tokens, each, count, inner, outer, dtype, codes, 0.1, "any")
