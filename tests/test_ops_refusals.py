"""What the convolution layers of ``ops`` and the block on them refuse, or answer without a launch: before anything
touches a device, so on the CPU. The kernels read as many weights as the input's channels ask for, so a wrong shape must
not reach them."""
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


@pytest.mark.parametrize("shape", [(0, 4, 4, 512), (2, 0, 4, 512), (2, 4, 0, 64)])
@pytest.mark.parametrize("f,ks", [(ops.conv2d, 1), (ops.conv2d, 3), (ops.conv2d_transpose, 3)])
def test_convolutions_of_no_pixels(f, ks, shape):
    """An empty batch is one (the choice of split counts divided by its blocks, which ended the process)."""
    C = shape[3]
    x = torch.zeros(shape, dtype=torch.bfloat16, requires_grad=True)
    w, b = torch.ones(ks, ks, C, C, requires_grad=True), torch.ones(C, requires_grad=True)
    y = f(x, w, b)
    assert y.shape == x.shape and y.dtype == x.dtype
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert gx.shape == x.shape and gw.shape == w.shape and not gw.any() and not gb.any()


def test_split_counts_of_no_pixels():
    from crack_detection_federatedlearning_grpc_amd._native_loader import hip
    assert hip().conv_splits(0, 4, 4, 512, 1, 1, 0, 512) == 1 and hip().conv_splits(0, 8, 8, 512, 3, 1, 1, 512) == 1
