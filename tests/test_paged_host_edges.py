"""Refusals of the paged-cache entry points beyond those of test_paged_host.py (no GPU is
needed for a refusal)."""

from __future__ import annotations

import pytest

from test_paged_host import CALLS, INVALID, cache, call, ptr


# ends and starts of one array inside another: a row of 2 x 4 heads of 128 fp32 values is 4096
# bytes, gathered state of 2 x 2 x 128 slots 2048
@pytest.mark.parametrize("name,change", [
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(3) + 2044)),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(3) - 4092)),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(4))),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(weight_out=ptr(1) - 2044)),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(1) + 4)),
    ("rtxllm_attn_decode_pages_gqa_f16", dict(out=ptr(1) + 60)),
    ("rtxllm_attn_decode_pages_gqa_f16", dict(out=ptr(2) - 4092)),
    ("rtxllm_kv_evict_f16", dict(weight_out=ptr(0) - 2044)),
    ("rtxllm_kv_evict_f16", dict(weight_out=ptr(1) + 4)),
    ("rtxllm_kv_evict_f16", dict(slot_pos_out=ptr(0) + 4)),
    ("rtxllm_kv_evict_f16", dict(slot_pos_out=ptr(1) - 2044)),
])
def test_outputs_inside_other_arrays(rlib, name, change):
    assert set(change) <= set(CALLS[name])
    assert call(rlib, name, cache(), **change) == INVALID
