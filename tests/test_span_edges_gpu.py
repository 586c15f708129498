"""Edges of the windowed and shared-prefix attention on the GPU, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import span_cases as S
import test_window_attention_gpu as T
from vllm_b200 import _native as N
from workloads import bf16_to_f32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pos0", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 30, 2 ** 31 - 64, 2 ** 30])
def test_prefill_positions_next_to_the_largest_are_reported(pos0):
    """A tile whose last position passes 32 bits writes nothing, as any position past the table."""
    case = S.SpanCase(93, [200, 64], kv_heads=2, window=50, sinks=2, q_counts=[30, 64])
    ok, _ = T.run_prefill(case)
    case.q_pos0[0] = pos0
    out = torch.full((94, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    got, err = T.run_prefill(case, out=out)
    assert err == N.TVP_DEVERR_BAD_TOKEN
    assert (bf16_to_f32(got[:30]) == 7.0).all() and np.array_equal(got[30:], ok[30:])
