"""Attention with the weights in one 16-bit part, as calls of many pairs have them, and in two, as calls of few: each
over the small shapes, whatever the number of pairs would choose (marked gpu)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from crack_detection_federatedlearning_grpc_amd import ops  # noqa: E402
from crack_detection_federatedlearning_grpc_amd._native_loader import hip  # noqa: E402
from test_gpu_block_ops import (  # noqa: E402, F401
    Exact,
    allowed,
    close,
    half_step,
    qkvg,
    test_attention_causal_ignores_the_future,
    test_attention_gradient_against_differences,
    test_attention_groups_do_not_hear_each_other,
    test_attention_ignores_what_is_not_allowed,
    test_attention_infinite_gradient_is_not_lost,
    test_attention_is_the_same_every_time,
    test_attention_lengths,
    test_attention_many_blocks,
    test_attention_mask_lengths_and_causal_together,
    test_attention_masked_rows_hear_nothing_of_a_bad_value,
    test_attention_masks,
    test_attention_matches_definition,
    test_attention_scale,
    test_attention_split_walks,
    test_attention_strides_and_alignment,
)


@pytest.fixture(params=["one", "two"], autouse=True)
def parts(request):
    hip().set_tune(hip().TUNE_ATTN_FINE, 1 if request.param == "one" else 2)
    yield request.param
    hip().set_tune(hip().TUNE_ATTN_FINE, 0)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_two_parts_round_the_output_once(D, dt, parts):
    """Values above zero, so that the output is as large as its terms. One part: u for the weights and u for the
    output, which out_tol counts; two parts leave 2 u^2 of the weights' u."""
    q, k, v, _ = qkvg(2, 90, 200, 4, 2, D, dt)
    v = v.abs()
    out = ops.attention(q, k, v)
    ex = Exact(q, k, v, None, allowed(2, 4, 90, 200, None, None, False), None)
    u = half_step(dt)
    close(out, ex.out, ex.out_tol - ((u - 2 * u * u) * ex.out if parts == "two" else 0), "out")
    few = ops.attention(q[:, :3], k, v)                          # few rows: always two parts
    close(few, ex.out[:, :3], ex.out_tol[:, :3] - (u - 2 * u * u) * ex.out[:, :3], "few rows")
