"""Refusals of the serving calls at the ends of what their numbers can be (CPU)."""
import pytest

from mimir_framework_b200 import abi, runtime as rt


@pytest.mark.parametrize("scale", [float("inf"), -float("inf")])
def test_a_scale_that_is_not_finite_is_refused(scale):
    cache = rt.paged_cache(k=16, v=16, type=abi.T_F16, n_pages=4, page_size=16, kv_heads=2, head_dim=64, page_stride=2048, slot_stride=128, head_stride=64)
    batch = rt.paged_batch(row_start=16, kv_len=16, page_table=16, table_stride=4, n_seqs=1, n_rows=1, max_rows=1, max_kv=64)
    att = rt.paged_attention(q=16, out=16, type=abi.T_F16, heads=4, row_stride=256, head_stride=64, out_row_stride=256, out_head_stride=64, scale=scale)
    for f in (lambda: rt.dev_paged_attention(cache, batch, att), lambda: rt.paged_attention_workspace(cache, batch, att)):
        with pytest.raises(rt.MimirB200Error, match="scale") as e:
            f()
        assert e.value.status == abi.E_INVALID


@pytest.mark.parametrize("magnitude", [1e39, 1e300, float("inf")])
def test_a_rotary_magnitude_beyond_fp32_is_refused(magnitude):
    with pytest.raises(rt.MimirB200Error, match="magnitude") as e:
        rt.rope_plan(64, magnitude=magnitude)
    assert e.value.status == abi.E_INVALID
