"""CPU: which kernel a linear forward call goes to (rules on sizes, types and alignment; both sides of each were timed), and that the GPU tests' sizes reach every one of them."""
import pytest

from simhand_amd import _lib
from tests.test_gpu_row_inplace import SHAPES
from tests.test_gpu_row_ops import SHAPES_LIN, SHAPES_MANY
from tests.test_gpu_row_rules import BORDERS

SKINNY, ROWS, TILES256, DMA, STAGED = range(5)
F32, H16 = 0, 1


def kernel(m, k, n, dtype=H16, aligned=1, residual=0):
    return _lib.load().simhand_test_linear_kernel(m, k, n, dtype, aligned, residual)


@pytest.mark.parametrize("m,k,n,residual,want", [
    # ragged rows with a residual: registers only where K is long and out is wide
    (200000, 129, 130, 1, STAGED), (361472, 33, 520, 1, STAGED), (503552, 333, 64, 1, STAGED), (2409472, 33, 50, 1, STAGED), (527616, 129, 250, 1, STAGED),
    (314880, 505, 130, 1, ROWS), (100000, 333, 777, 1, ROWS), (40000, 505, 777, 1, ROWS), (443392, 201, 250, 1, ROWS),
    # without one: from three units a row tile
    (300000, 77, 192, 0, ROWS), (100000, 333, 777, 0, ROWS), (200000, 129, 130, 0, STAGED),
    # whole chunks
    (100352, 512, 2048, 1, ROWS), (1605632, 128, 512, 1, ROWS), (568064, 32, 320, 1, ROWS), (401408, 256, 1024, 0, ROWS), (347136, 256, 320, 0, ROWS),
    (446208, 256, 192, 0, TILES256), (1605632, 128, 512, 0, TILES256), (624896, 256, 64, 0, DMA),
    # few rows, few tiles
    (64, 512, 128, 0, SKINNY), (65, 512, 128, 0, DMA), (5001, 1000, 333, 0, DMA), (5001, 1001, 333, 0, STAGED)])
def test_rule(m, k, n, residual, want):
    assert kernel(m, k, n, residual=residual) == want


def test_the_types_and_the_alignment():
    assert kernel(401408, 256, 1024, F32) == DMA and kernel(401408, 257, 1024, F32) == STAGED
    assert kernel(401408, 256, 1024, aligned=0) == ROWS and kernel(401408, 1024, 256, aligned=0) == STAGED


def test_a_workspace_is_asked_for_wherever_one_is_needed():
    """The query knows no residual: it has to cover the call with and without one."""
    lib = _lib.load()
    for k in (33, 45, 129, 191, 192, 201, 256, 333, 505, 512, 513):
        for n in (50, 64, 127, 128, 130, 191, 192, 256, 777, 4096, 4097):
            for m in (1000, 16384, 131072, 400000):
                for aligned in (0, 1):
                    ragged = k % 8 != 0 or not aligned
                    if ragged and any(kernel(m, k, n, H16, aligned, r) == ROWS for r in (0, 1)):
                        assert lib.simhand_linear_fwd_workspace_bytes(m, k, n, H16, aligned) >= n * ((k + 7) // 8 * 8) * 2, (m, k, n, aligned)


def test_the_gpu_tests_reach_every_kernel():
    for residual in (0, 1):
        seen = {kernel(*s, residual=residual) for s in SHAPES_LIN + SHAPES_MANY}
        assert seen == {SKINNY, ROWS, TILES256, DMA, STAGED}
    assert {kernel(*s, residual=1) for s in SHAPES} == {SKINNY, ROWS, TILES256, DMA, STAGED}
    steps = lambda rag, res: {(k + 127) // 128 for m, k, n in SHAPES_LIN + SHAPES_MANY + SHAPES + BORDERS if kernel(m, k, n, residual=res) == ROWS and (k % 8 != 0) == rag}  # noqa: E731
    assert steps(False, 1) == {1, 2, 3, 4} and steps(True, 1) == {2, 3, 4} and steps(False, 0) == {2, 3, 4} and steps(True, 0) == {1, 2, 3, 4}
