"""Edges of the windowed and shared-prefix attention on the GPU, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import span_cases as S
import test_shared_prefix_gpu as P
import test_window_attention_gpu as T
from vllm_b200 import _native as N
from vllm_b200 import ops
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


def many(rng, n, rows_hi, pages_hi):
    """Groups of 0 to rows_hi rows behind 0 to pages_hi pages."""
    return [(int(r), int(p)) for r, p in zip(rng.integers(0, rows_hi + 1, n), rng.integers(0, pages_hi + 1, n))]


@pytest.mark.parametrize("n", [31, 32, 33, 191, 192, 193, 1023, 1024, 1025, 2100])
def test_many_groups(n):
    """Around the number of groups that a warp's lanes hold, and the plan's block."""
    rng = np.random.default_rng(n)
    groups = many(rng, n, 3 if n < 1000 else 1, 5 if n < 1000 else 2)
    groups[0], groups[-1] = (2, 7), (1, 3)
    case = S.SpanCase(n, P.rows(rng, groups, 40), groups=groups, kv_heads=1)
    got, err = P.run(case)
    assert err == 0
    S.check(got, case)
    again, err = P.run(case)
    assert err == 0 and np.array_equal(got, again)


@pytest.mark.parametrize("n", [33, 192, 193])
@pytest.mark.parametrize("ctas", [0, 300])
def test_prefixes_of_many_groups_cut_into_pieces(n, ctas):
    """Fewer streams than CTAs: long prefixes take several pieces each, with empty groups between."""
    rng = np.random.default_rng(n)
    groups = [(1, int(p)) if i % 3 else (0, 9) for i, p in enumerate(rng.integers(0, 90, n))]
    case = S.SpanCase(200 + n, P.rows(rng, groups, 60), groups=groups, kv_heads=2)
    got, err = P.run(case, num_ctas=ctas)
    assert err == 0
    S.check(got, case)


@pytest.mark.parametrize("n", [50, 210])
def test_faults_of_many_groups_are_reported(n):
    rng = np.random.default_rng(9)
    groups = [(2, 2)] * n
    case = S.SpanCase(60, P.rows(rng, groups, 60), groups=groups, kv_heads=2)
    rows = case.group_rows.copy()
    rows[44] = 2 * n + 1
    got, err = P.run(case, group_rows=rows)
    assert err == N.TVP_DEVERR_BAD_PLAN and (bf16_to_f32(got) == 3.0).all()
    for pages in (-1, 1 << 20):
        bad = case.prefix_pages.copy()
        bad[40] = pages
        got, err = P.run(case, prefix_pages=bad)
        assert err & N.TVP_DEVERR_BAD_LENGTH
        # (not bit for bit: that group's own pages move where the other rows are cut)
        others = np.r_[0:80, 82:2 * n]
        want, tol = case.oracle()
        assert (np.abs(bf16_to_f32(got[others]) - want[others]) <= tol[others]).all()


def test_one_workspace_for_few_groups_and_many():
    ws = ops.SpanWorkspace(500, "cuda", kv_heads=2, max_groups=250)
    for i, n in enumerate((250, 3, 193, 192, 250)):
        rng = np.random.default_rng(n)
        groups = many(rng, n, 2, 9)
        groups[0] = (1, 4)
        case = S.SpanCase(300 + i, P.rows(rng, groups, 50), groups=groups, kv_heads=2)
        got, err = P.run(case, workspace=ws)
        assert err == 0
        S.check(got, case)
