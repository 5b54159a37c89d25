"""More tiles than a launch takes are refused before anything is launched, on the CPU: where coding x came first, these calls
would end in the runtime's error and not in their own."""
import ctypes

import pytest

from test_blocks_args import P, rejected

MOST = (1 << 31) - 1


def workspace(query, *sizes):
    from tcc_spmm_amd._lib import check, lib
    size = ctypes.c_size_t()
    check(getattr(lib(), query)(*sizes, ctypes.byref(size)))
    return size.value


# type, format, rows, inner, outer: FP32 of 8-bit rows in tiles of 64, all others of 256 in a launch of fewer than 2^24.
@pytest.mark.parametrize("t,form,rows,inner,outer", [(0, 0, 1 << 30, 1, 1), (0, 0, 1 << 24, 128, 4096), (1, 0, MOST, 1, 512),
                                                     (2, 1, MOST, 130, 512), (0, 1, 1 << 22, 64, 1 << 18)])
@pytest.mark.parametrize("keep", [False, True])
def test_linear_micro(t, form, rows, inner, outer, keep):
    from tcc_spmm_amd._lib import lib
    keep = P if keep and not form else None
    size = workspace("tcc_linear_micro_workspace", rows, inner, outer, t, form, keep is not None)
    rejected(lib().tcc_linear_micro(P, inner, t, form, P, P, None, P, outer, keep, keep, rows, inner, outer, P, size, None),
             b"linear micro: more tiles than a launch takes")


@pytest.mark.parametrize("t,form,choices,each,inner,outer", [(0, 0, 1 << 30, 1, 1, 1), (1, 0, MOST, 1, 1, 512),
                                                             (2, 1, 1 << 30, 4, 1, 1024)])
def test_linear_experts(t, form, choices, each, inner, outer):
    from tcc_spmm_amd._lib import lib
    for by_token in (0, 1):
        size = workspace("tcc_linear_experts_workspace", choices, each, 4, by_token, inner, outer, t, form)
        call = lib().tcc_linear_experts(P, inner, t, form, by_token, P, P, None, P, outer, P, P, choices, each, 4, inner, outer,
                                        P, size, None)
        # tokens' codes are reached by 32 bits: of one too many rows for that the call says so
        rejected(call, b"gather them" if by_token and choices // each * (64 if form else 128) >> 31 else
                 b"linear experts: more tiles than a launch takes")


@pytest.mark.parametrize("t,rows,inner,outer", [(0, MOST, 600, 512), (1, MOST, 600, 512), (2, 1 << 24, 600, 1 << 18)])
@pytest.mark.parametrize("keep", [False, True])
def test_linear_blocks(t, rows, inner, outer, keep):
    from tcc_spmm_amd._lib import lib
    size = workspace("tcc_linear_blocks_workspace", rows, inner, outer, t, keep)
    keep = P if keep else None
    rejected(lib().tcc_linear_blocks(P, inner, t, P, P, None, P, outer, keep, keep, rows, inner, outer, P, size, None),
             b"linear blocks: more tiles than a launch takes")
