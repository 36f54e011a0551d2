"""CPU: the relative position bias under a default device.  The bucket borders are kept on the host from one call to the next."""
import pytest
import torch

from openvis_amd import ops


def _meta(*shape):
    return torch.empty(*shape, dtype=torch.float32, device="meta")


@pytest.mark.parametrize("both", [True, False])
def test_a_default_device_does_not_move_the_borders(both):
    with torch.device("meta"):                                    # as torch.set_default_device("cuda") would: factories make tensors there
        assert ops.relpos_bias_1d(_meta(42, 4), 3, 9, bidirectional=both).shape == (4, 3, 9)
        assert ops.relpos_bias_1d_backward(_meta(2, 4, 3, 9), 44, bidirectional=both).shape == (44, 4)
    assert ops.relpos_bias_1d(_meta(42, 4), 3, 9, bidirectional=both).shape == (4, 3, 9)
    assert ops.relpos_bias_1d_backward(_meta(2, 4, 3, 9), 44, bidirectional=both).shape == (44, 4)


def test_a_call_under_fake_tensors_leaves_nothing_behind():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        try:
            ops.relpos_bias_1d(mode.from_tensor(_meta(46, 4)), 3, 9)
        except RuntimeError:
            pass                                                  # whether such a call is served is another matter
    assert ops.relpos_bias_1d(_meta(46, 4), 3, 9).shape == (4, 3, 9)


def test_inference_mode():
    with torch.inference_mode():
        assert ops.relpos_bias_1d(_meta(50, 4), 3, 9).shape == (4, 3, 9)
    assert ops.relpos_bias_1d(_meta(50, 4), 3, 9).shape == (4, 3, 9)
