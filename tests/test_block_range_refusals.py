"""Calls of the operators around a transformer's blocks that lie beyond their ranges though they have no rows. No GPU: the tensors only carry addresses."""
import pytest


@pytest.mark.parametrize("cols", [1 << 29, 1 << 31, (1 << 32) + 8])
def test_gradient_of_no_rows_that_are_too_long(hpt, cols):
    """The gradient of gamma would be zeros, of more columns than the kernels count."""
    at = lambda shape, place: hpt.Tensor.from_raw(place << 40, shape, hpt.f32)  # noqa: E731
    x = at([0, cols], 1)
    with pytest.raises(hpt.ShapeError, match="fewer than"):
        x.rms_norm_backward(at([0, cols], 2), [cols], out=at([0, cols], 3), gamma_out=at([cols], 4))
    with pytest.raises(hpt.ShapeError, match="fewer than"):
        hpt.rms_norm_backward_workspace(x, 1)
    assert hpt.rms_norm_backward_workspace(at([0, (1 << 29) - 1], 1), 1) == 0
