"""Kernel choice of the grouped products (mxb_grouped_plan_for), host-only, on a 148-SM GPU.  The launches use the same
function, so these cases pin what runs."""
import ctypes as C

import pytest

from minixla_b200 import lib as mlib

FORWARD, GRAD_A, GRAD_B = mlib.MXB_GROUPED_FORWARD, mlib.MXB_GROUPED_GRAD_A, mlib.MXB_GROUPED_GRAD_B
SINGLE, PAIR = mlib.MXB_KERNEL_SINGLE_CTA, mlib.MXB_KERNEL_CTA_PAIR

# (product, rows, groups, N, K) -> (kernel, tile_rows, tile_cols, k_splits)
CASES = [
    ((FORWARD, 2, 8, 4096, 1024), (SINGLE, 64, 128, 2)),       # 64 tiles at most: two CTAs for each
    ((FORWARD, 128, 64, 2048, 1024), (SINGLE, 64, 128, 1)),
    ((FORWARD, 8192, 8, 4096, 4096), (PAIR, 256, 256, 1)),
    ((GRAD_A, 4001, 16, 4096, 1024), (PAIR, 256, 256, 1)),
    ((GRAD_B, 8191, 8, 4096, 1024), (PAIR, 256, 256, 1)),
    ((FORWARD, 672, 8, 4096, 2048), (SINGLE, 64, 128, 1)),     # 84 rows a group
    ((FORWARD, 680, 8, 4096, 2048), (PAIR, 256, 256, 1)),      # 85
    ((GRAD_A, 459, 12, 1022, 811), (SINGLE, 64, 128, 1)),
    ((FORWARD, 32768, 4, 128, 1024), (SINGLE, 64, 128, 1)),    # results too narrow for a pair
    ((GRAD_B, 8192, 1, 512, 512), (SINGLE, 128, 128, 8)),      # 16 tiles
    ((GRAD_B, 16384, 8, 256, 256), (SINGLE, 128, 128, 4)),
    ((GRAD_B, 4096, 8, 1024, 64), (SINGLE, 128, 128, 2)),
    ((FORWARD, 130, 5, 64, 512), (SINGLE, 64, 128, 8)),
]


@pytest.mark.parametrize("args,want", CASES, ids=lambda v: "x".join(map(str, v)))
def test_plan(args, want):
    p = mlib.grouped_plan(*args)
    assert (p.kernel, p.tile_rows, p.tile_cols, p.k_splits) == want and p.products == args[2]


@pytest.mark.parametrize("args", [(-1, 4, 2, 8, 8, 148), (3, 4, 2, 8, 8, 148), (0, 0, 2, 8, 8, 148), (0, 4, 0, 8, 8, 148),
                                  (0, 4, 1025, 8, 8, 148), (0, 4, 2, 0, 8, 148), (0, 4, 2, 8, 0, 148), (0, 4, 2, 8, 8, 1),
                                  (0, 2 ** 30 + 1, 2, 8, 8, 148)], ids=str)
def test_refusals(lib, args):
    assert lib.mxb_grouped_plan_for(*args, C.byref(mlib.GemmPlan())) == mlib.MXB_E_ARG
    assert "mxb_grouped_plan_for" in mlib.last_error()


def test_refuses_no_plan(lib):
    assert lib.mxb_grouped_plan_for(0, 4, 2, 8, 8, 148, None) == mlib.MXB_E_ARG
