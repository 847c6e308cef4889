"""The classifier head without a GPU: calls at the ends of what its arguments can hold."""
import ctypes

import pytest

UNSUPPORTED, WORKSPACE = 2, 3
MOST = 2 ** 31 - 65536


def calls(rows, features, classes, dtype):
    """Status of the forward and the backward call, without a workspace: nothing is launched."""
    from deformable_kernels import _cabi as C
    one, null = ctypes.c_void_p(16), ctypes.c_void_p(0)
    forward = C.lib.dk_linear_cross_entropy_forward(one, one, null, one, one, null, rows, features, classes, -100, 1, 0.0, dtype, null, 0, null)
    backward = C.lib.dk_linear_cross_entropy_backward(one, one, one, null, one, one, one, one, null, rows, features, classes, -100, 1, 0.0,
                                                      dtype, null, 0, null)
    return forward, backward


@pytest.mark.parametrize("dtype", range(4))
@pytest.mark.parametrize("which", range(3))
def test_sizes_whose_loops_would_pass_32_bits_are_refused(which, dtype):
    from deformable_kernels import _cabi as C
    for size in (2 ** 31 - 1, MOST + 1):
        sizes = [1, 1, 1]
        sizes[which] = size
        assert calls(*sizes, dtype) == (UNSUPPORTED, UNSUPPORTED)
        for q in (C.lib.dk_linear_cross_entropy_forward_workspace_bytes, C.lib.dk_linear_cross_entropy_backward_workspace_bytes):
            assert q(*sizes, dtype) == 0
    if which == 2:
        assert calls(1, 1, MOST, dtype)[0] == WORKSPACE


@pytest.mark.parametrize("dtype", range(4))
def test_more_logits_than_a_plan_can_count_are_refused(dtype):
    for rows, classes in ((MOST, MOST), (2 ** 30, 2 ** 27)):
        assert calls(rows, 1, classes, dtype) == (UNSUPPORTED, UNSUPPORTED)


@pytest.mark.parametrize("dtype", range(4))
def test_many_features_are_no_reason_to_refuse(dtype):
    """No sum stays in one accumulator for longer than a wait may take."""
    assert calls(8, 2 ** 28, 2, dtype) == (WORKSPACE, WORKSPACE)


def test_dropout_does_not_write_the_state_that_it_reads():
    from deformable_kernels import _cabi as C
    at = ctypes.c_void_p
    for state, used in ((64, 64), (64, 72), (64, 56)):
        assert C.lib.dk_dropout(at(1024), at(2048), 8, 1, 0.5, 0, 0, at(state), at(used), 0, at(0)) == 1
