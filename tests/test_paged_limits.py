"""The limits that include/sa_cuda.h gives for the paged operators' numbers, on
both sides: what is refused on the CPU, and results just inside on the GPU."""
import pytest
import torch

from test_paged_args import P, _decode, _kv, _prefill, _prefix, _refused

# largest fp32 whose product with fp32 log2(e) = 0x1.715476p+0 is finite, and the next one
SCALE_MAX, SCALE_OVER = float.fromhex("0x1.62e42ep+127"), float.fromhex("0x1.62e430p+127")


@pytest.mark.parametrize("call", [_decode, _prefill, _prefix])
def test_scales_that_log2e_takes_past_fp32_are_refused(call):
    log2e = torch.tensor(1.4426950408889634)
    assert torch.isfinite(torch.tensor(SCALE_MAX) * log2e) and torch.isinf(torch.tensor(SCALE_OVER) * log2e)
    for scale in (SCALE_OVER, 3.0e38, float("inf")):
        _refused(call(_kv(), scale=scale), "scale")
    _refused(call(_kv(), scale=SCALE_MAX), "ctx is NULL")          # taken: the next check's error
