"""The 8-bit cache's tests that compare values by their bounds alone, with a check that
takes no NaN: caches start as NaN wherever nothing has been written, so stale codes,
scales and weights that reach a result show up as one."""
import pytest

import test_gpu_kv8 as kv8
from test_gpu_kv8 import (  # noqa: F401  (collected here with their parameters)
    test_a_serving_run, test_behind_the_projections, test_decode_long_many_splits,
    test_decode_rows_of_many_lengths, test_decode_scales_of_q,
    test_decode_values_of_very_different_blocks, test_evict_then_append_and_attend,
    test_nan_and_inf_stay_where_they_are, test_offsets_past_32_bits, test_prefill_long,
    test_prefill_scales_of_q, test_prefill_weights_in_several_launches,
    test_prefill_weights_long, test_weights_accumulate)
import kv8_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setattr(kv8, "check_rows", ref.check_rows)
