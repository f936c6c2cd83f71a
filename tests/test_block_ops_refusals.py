"""What attention, rotary positions and layer norm refuse: checked before anything touches a device, so on the CPU."""
import math

import pytest
import torch

from crack_detection_federatedlearning_grpc_amd import ops

BF = torch.bfloat16


def z(*shape, dt=BF):
    return torch.zeros(*shape, dtype=dt)


Q, KV = z(2, 5, 4, 32), z(2, 7, 2, 32)


@pytest.mark.parametrize("err,args,kw", [
    (ValueError, (z(5, 4, 32), KV, KV), {}),                                  # axes
    (TypeError, (z(2, 5, 4, 32, dt=torch.float32), KV, KV), {}),              # type
    (TypeError, (Q, KV.half(), KV), {}),                                      # mixed types
    (ValueError, (Q, KV, z(2, 8, 2, 32)), {}),                                # k and v apart
    (ValueError, (Q, z(3, 7, 2, 32), z(3, 7, 2, 32)), {}),                    # images
    (ValueError, (Q, z(2, 7, 2, 64), z(2, 7, 2, 64)), {}),                    # channels
    (ValueError, (z(2, 5, 4, 20), z(2, 7, 2, 20), z(2, 7, 2, 20)), {}),       # channels not in eights
    (ValueError, (z(2, 5, 4, 136), z(2, 7, 2, 136), z(2, 7, 2, 136)), {}),    # too many channels
    (ValueError, (z(2, 5, 4, 0), z(2, 7, 2, 0), z(2, 7, 2, 0)), {}),
    (ValueError, (Q, z(2, 7, 3, 32), z(2, 7, 3, 32)), {}),                    # heads that do not divide
    (ValueError, (Q, z(2, 7, 0, 32), z(2, 7, 0, 32)), {}),
    (TypeError, (Q, KV, KV), {"mask": torch.zeros(5, 7)}),                    # additive masks
    (ValueError, (Q, KV, KV), {"mask": torch.zeros(7, 5, dtype=torch.bool)}),
    (ValueError, (Q, KV, KV), {"mask": torch.zeros(1, 2, 4, 5, 7, dtype=torch.bool)}),
    (ValueError, (Q, KV, KV), {"mask": torch.zeros(2, 2, 5, 7, dtype=torch.bool)}),   # of the key heads
    (TypeError, (Q, KV, KV), {"lengths": torch.tensor([7, 7])}),              # int64
    (ValueError, (Q, KV, KV), {"lengths": torch.tensor([7], dtype=torch.int32)}),
    (ValueError, (Q, KV, KV), {"scale": 0.0}),
    (ValueError, (Q, KV, KV), {"scale": -1.0}),
    (ValueError, (Q, KV, KV), {"scale": math.nan}),
    (RuntimeError, (Q, KV, KV), {}),                                          # host tensors
])
def test_attention_refuses(err, args, kw):
    with pytest.raises(err):
        ops.attention(*args, **kw)


@pytest.mark.parametrize("err,args", [
    (ValueError, (z(5, 4, 32), 2)), (ValueError, (z(2, 5, 7, 32), 2)), (ValueError, (z(2, 5, 6, 32), 4, 2)),
    (ValueError, (z(2, 5, 6, 32), 0)), (ValueError, (z(2, 5, 9, 32), 5, 2)), (RuntimeError, (z(2, 5, 6, 32), 2))])
def test_attention_qkv_refuses(err, args):
    with pytest.raises(err):
        ops.attention_qkv(*args)


@pytest.mark.parametrize("err,x,kw", [
    (ValueError, z(()), {}), (TypeError, z(3, 4, dt=torch.float64), {}), (TypeError, z(3, 4, dt=torch.int32), {}),
    (ValueError, z(3, 0), {}), (ValueError, z(1, 8193), {}), (ValueError, z(3, 4), {"eps": -1.0}),
    (ValueError, z(3, 4), {"eps": math.inf}), (TypeError, z(3, 4), {"weight": z(4)}),
    (ValueError, z(3, 4), {"weight": z(3, dt=torch.float32)}), (ValueError, z(3, 4), {"bias": z(1, 4, dt=torch.float32)}),
    (RuntimeError, z(3, 4), {})])
def test_layer_norm_refuses(err, x, kw):
    with pytest.raises(err):
        ops.layer_norm(x, **kw)


POS = torch.zeros(2, 5, dtype=torch.int32)


@pytest.mark.parametrize("err,x,pos,dims,kw", [
    (ValueError, z(5, 4, 32), POS, (16, 16), {}), (TypeError, z(2, 5, 4, 32, dt=torch.float64), POS, (16, 16), {}),
    (ValueError, z(2, 5, 4, 32), POS, (), {}), (ValueError, z(2, 5, 4, 32), POS, (2,) * 5, {}),
    (ValueError, z(2, 5, 4, 32), POS, (15, 17), {}), (ValueError, z(2, 5, 4, 32), POS, (-2, 16), {}),
    (ValueError, z(2, 5, 4, 32), POS, (0, 0), {}), (ValueError, z(2, 5, 4, 32), POS, (16, 18), {}),
    (ValueError, z(2, 5, 4, 32), POS, (32,), {}), (ValueError, z(2, 6, 4, 32), POS, (16, 16), {}),
    (ValueError, z(2, 5, 4, 32), torch.zeros(2, 3, 5, dtype=torch.int32), (16, 16), {}),
    (TypeError, z(2, 5, 4, 32), POS.double(), (16, 16), {}), (TypeError, z(2, 5, 4, 32), POS.short(), (16, 16), {}),
    (ValueError, z(2, 5, 4, 32), POS, (16, 16), {"theta": 0.0}),
    (ValueError, z(2, 5, 4, 32), POS, (16, 16), {"theta": math.nan}),
    (ValueError, z(2, 5, 4, 32), torch.zeros(2, 5, requires_grad=True), (16, 16), {}),
    (RuntimeError, z(2, 5, 4, 32), POS, (16, 16), {})])
def test_rotary_refuses(err, x, pos, dims, kw):
    with pytest.raises(err):
        ops.rotary(x, pos, dims, **kw)


@pytest.mark.parametrize("sizes", [(), (0, 3), (2.5,), (-1,)])
def test_grid_positions_refuses(sizes):
    with pytest.raises(ValueError):
        ops.grid_positions(*sizes)


@pytest.mark.parametrize("kw", [{"x": z(4, 4, 64)}, {"w_qkv": torch.zeros(1, 1, 64, 100)}, {"heads": 0},
                                {"w_out": torch.zeros(1, 1, 64, 64)}, {"kv_heads": 3},
                                {"w_qkv": torch.zeros(1, 1, 64, 12 * 20)}])
def test_self_attention2d_refuses(kw):
    base = {"x": z(1, 4, 4, 64), "norm_weight": torch.ones(64), "norm_bias": torch.zeros(64),
            "w_qkv": torch.zeros(1, 1, 64, 12 * 32), "w_out": torch.zeros(1, 1, 128, 64), "heads": 4}
    with pytest.raises(ValueError):
        ops.self_attention2d(**{**base, **kw})


@pytest.mark.parametrize("scale", [1e-50, 3e38, 1e39, math.inf])
def test_attention_refuses_scales_outside_float32(scale):
    with pytest.raises(ValueError, match="float32"):
        ops.attention(Q, KV, KV, scale=scale)
