"""What the convolution layers of ``ops`` and the block on them refuse: checked before anything touches a device, so on
the CPU. The kernels read as many weights as the input's channels ask for, so a wrong shape must not reach them."""
import pytest
import torch

from crack_detection_federatedlearning_grpc_amd import ops

X = torch.zeros(1, 4, 4, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("f,x,w,b", [
    (ops.conv2d, X, torch.zeros(1, 1, 32, 64), None), (ops.conv2d, X, torch.zeros(3, 3, 32, 64), None),
    (ops.conv2d, X, torch.zeros(1, 1, 96, 64), None), (ops.conv2d_transpose, X, torch.zeros(3, 3, 64, 32), None),
    (ops.conv2d, X[0], torch.zeros(1, 1, 64, 64), None), (ops.conv2d, X, torch.zeros(1, 64, 64), None),
    (ops.conv2d, X, torch.zeros(1, 1, 64, 64), torch.zeros(32)),
    (ops.conv2d_transpose, X, torch.zeros(3, 3, 32, 64), torch.zeros(64)),
    (ops.conv2d, X, torch.zeros(1, 1, 64, 64, device="meta"), None)])
def test_convolutions_refuse_weights_of_other_shapes(f, x, w, b):
    with pytest.raises(ValueError):
        f(x, w, b)


@pytest.mark.parametrize("kw", [
    {"w_qkv": torch.zeros(1, 1, 32, 12 * 32)}, {"w_qkv": torch.zeros(3, 3, 64, 12 * 32)},
    {"w_out": torch.zeros(1, 1, 128, 32)}, {"w_out": torch.zeros(3, 3, 128, 64)}])
def test_self_attention2d_refuses_weights_of_other_shapes(kw):
    base = {"x": X, "norm_weight": torch.ones(64), "norm_bias": torch.zeros(64),
            "w_qkv": torch.zeros(1, 1, 64, 12 * 32), "w_out": torch.zeros(1, 1, 128, 64), "heads": 4}
    with pytest.raises(ValueError):
        ops.self_attention2d(**{**base, **kw})
