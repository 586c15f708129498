"""Causal prefill attention with positions that pass its table's: reported, nothing written."""
import numpy as np
import pytest
import torch

from gpu_util import dev_bf16, dev_i32, host_bf16
from test_prefill_gpu import make_case, run_prefill
from vllm_b200 import _native as N
from vllm_b200 import ops
from workloads import bf16_to_f32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 64, 2 ** 30, 190, -1])
def test_positions_past_the_table(first):
    case, q, cu_q, pos0 = make_case(93, [30, 64], context=[170, 0])
    ok, err = run_prefill(case, q, cu_q, pos0)
    assert err == 0
    pos0 = pos0.copy()
    pos0[0] = first
    err, qd = ops.new_error_word("cuda"), dev_bf16(q)
    out = torch.full_like(qd, 7.0)
    ops.paged_prefill_attention(qd, dev_bf16(case.k_pool), dev_bf16(case.v_pool), 0, dev_i32(case.tables),
                                dev_i32(cu_q), dev_i32(pos0), 64, out=out, error=err)
    torch.cuda.synchronize()
    got = host_bf16(out)
    assert int(err.item()) == N.TVP_DEVERR_BAD_TOKEN
    assert (bf16_to_f32(got[:30]) == 7.0).all() and np.array_equal(got[30:], ok[30:])
