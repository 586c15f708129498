"""Decode attention of rows that share a prefix, on the GPU, against the 64-bit
oracle; NaN in every unused slot, -1 in the rows' entries of shared pages."""
import numpy as np
import pytest
import torch

import span_cases as S
from gpu_util import dev_bf16, dev_i32, host_bf16
from vllm_b200 import _native as N
from vllm_b200 import ops

pytestmark = pytest.mark.gpu


def run(case, num_ctas=0, workspace=None, group_rows=None, prefix_pages=None):
    err = ops.new_error_word("cuda")
    groups = len(case.prefix_pages)
    ws = workspace or ops.SpanWorkspace(len(case.lens), "cuda", num_ctas=num_ctas, kv_heads=case.kv_heads,
                                        max_groups=groups)
    q = dev_bf16(case.q)
    out = torch.full_like(q, 3.0)
    ops.paged_shared_prefix_decode_attention(
        q, dev_bf16(case.k_pool), dev_bf16(case.v_pool), case.layer, dev_i32(case.tables), dev_i32(case.lens),
        dev_i32(case.prefix_tables), dev_i32(case.prefix_pages if prefix_pages is None else prefix_pages),
        dev_i32(case.group_rows if group_rows is None else group_rows), ws, scale=case.scale, out=out, error=err)
    torch.cuda.synchronize()
    return host_bf16(out), int(err.item())


def rows(rng, groups, hi):
    """Lengths of the groups' rows: each group's prefix and 0..hi tokens more."""
    return np.concatenate([p * 16 + rng.integers(0, hi + 1, n) for n, p in groups] + [np.zeros(0, np.int64)])


@pytest.mark.parametrize("groups", [[(1, 1)], [(4, 3)], [(31, 2)], [(32, 5)], [(33, 4)], [(70, 9)],
                                    [(3, 2), (5, 7), (1, 1)], [(2, 0), (3, 4)], [(40, 3), (40, 11), (2, 6)]], ids=str)
def test_groups(groups):
    case = S.SpanCase(7 + len(groups), rows(np.random.default_rng(1), groups, 90), groups=groups)
    got, err = run(case)
    assert err == 0
    S.check(got, case, str(groups))


@pytest.mark.parametrize("kv_heads", [1, 2, 4, 8])
@pytest.mark.parametrize("ctas", [1, 5, 148, 400])
def test_any_heads_and_grid(kv_heads, ctas):
    groups = [(9, 21), (36, 13)]
    case = S.SpanCase(17, rows(np.random.default_rng(2), groups, 300), groups=groups, kv_heads=kv_heads, num_layers=2,
                      layer=1)
    got, err = run(case, num_ctas=ctas)
    assert err == 0
    S.check(got, case)


def test_rows_that_end_with_the_prefix_and_padded_rows():
    """Rows whose whole context is the prefix, and empty rows inside a group: zeros, no error."""
    groups = [(6, 4), (3, 2)]
    case = S.SpanCase(23, [64, 0, 65, 64, 0, 80, 0, 32, 33], groups=groups)
    got, err = run(case)
    assert err == 0
    S.check(got, case)
    assert (got[[1, 4, 6]] == 0).all()


def test_a_group_of_padded_rows_only():
    case = S.SpanCase(24, [0, 0, 0, 50], groups=[(3, 0), (1, 1)])
    got, err = run(case)
    assert err == 0
    S.check(got, case)


def test_rows_outside_every_group():
    groups = [(3, 4), (2, 1)]
    case = S.SpanCase(25, [70, 64, 100, 17, 16, 33, 0, 500], groups=groups)
    got, err = run(case)
    assert err == 0
    S.check(got, case)


def test_no_groups_is_plain_decode():
    case = S.SpanCase(26, [70, 1, 0, 300], groups=[])
    case.prefix_tables = np.full((1, 1), -1, np.int32)
    got, err = run(case)
    assert err == 0
    S.check(got, case)


def test_long_prefix_many_pieces_repeat_bit_for_bit():
    groups = [(5, 260)]
    case = S.SpanCase(27, rows(np.random.default_rng(3), groups, 400), groups=groups, kv_heads=2)
    ws = ops.SpanWorkspace(5, "cuda", kv_heads=2, max_groups=1)
    ref, err = run(case, workspace=ws)
    assert err == 0
    S.check(ref, case)
    for _ in range(10):
        got, err = run(case, workspace=ws)
        assert err == 0 and np.array_equal(got, ref)


def test_wide_scores():
    """Maxima that differ by hundreds between a prefix's pieces and the rows' own pages."""
    groups = [(12, 40)]
    case = S.SpanCase(28, rows(np.random.default_rng(4), groups, 200), groups=groups, kv_heads=2, scale=0.3)
    got, err = run(case)
    assert err == 0
    S.check(got, case)


def test_rows_shorter_than_their_prefix_are_reported():
    groups = [(4, 4)]
    lens = [70, 64, 90, 100]
    case = S.SpanCase(29, lens, groups=groups)
    ok, _ = run(case)
    case.lens[1] = 40
    got, err = run(case)
    assert err == N.TVP_DEVERR_BAD_LENGTH
    assert (got[1] == 0).all() and np.array_equal(got[[0, 2, 3]], ok[[0, 2, 3]])


def test_bad_pages_are_reported():
    groups = [(4, 4)]
    case = S.SpanCase(30, [70, 64, 90, 100], groups=groups)
    ok, _ = run(case)
    case.tables[2, 5] = case.num_pages
    got, err = run(case)
    assert err == N.TVP_DEVERR_BAD_PAGE and np.array_equal(got[[0, 1, 3]], ok[[0, 1, 3]])
    case.prefix_tables[0, 1] = -1
    got, err = run(case)
    assert err == N.TVP_DEVERR_BAD_PAGE
    assert np.isfinite(S.W.bf16_to_f32(got)).all()


@pytest.mark.parametrize("group_rows", [[0, 5, 3], [-1, 2, 4], [0, 2, 9], [3, 2, 4]])
def test_group_rows_out_of_order_write_nothing(group_rows):
    case = S.SpanCase(31, [70, 64, 40, 50], groups=[(2, 2), (2, 1)])
    got, err = run(case, group_rows=np.array(group_rows, np.int32))
    assert err == N.TVP_DEVERR_BAD_PLAN
    assert (S.W.bf16_to_f32(got) == 3.0).all()


@pytest.mark.parametrize("pages", [-1, 1 << 20])
def test_prefix_pages_out_of_range_are_reported(pages):
    case = S.SpanCase(32, [70, 64, 40, 50], groups=[(2, 2), (2, 1)])
    got, err = run(case, prefix_pages=np.array([2, pages], np.int32))
    assert err & N.TVP_DEVERR_BAD_LENGTH
    ok, _ = run(case)
    assert np.array_equal(got[:2], ok[:2])


def test_captured_and_replayed():
    groups = [(20, 30), (4, 3)]
    case = S.SpanCase(33, rows(np.random.default_rng(5), groups, 100), groups=groups)
    args = [dev_bf16(case.q), dev_bf16(case.k_pool), dev_bf16(case.v_pool), 0, dev_i32(case.tables),
            dev_i32(case.lens), dev_i32(case.prefix_tables), dev_i32(case.prefix_pages), dev_i32(case.group_rows)]
    ws, err, out = ops.SpanWorkspace(24, "cuda", max_groups=2), ops.new_error_word("cuda"), torch.empty_like(args[0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.paged_shared_prefix_decode_attention(*args, ws, out=out, error=err)
    side.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of one workspace, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.paged_shared_prefix_decode_attention(*args, ws, out=out, error=err)
        graphs.append(graph)
    for graph in graphs * 3:
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        S.check(host_bf16(out), case)


def test_many_small_groups():
    """More groups than a warp has lanes, some without a prefix or without rows."""
    rng = np.random.default_rng(6)
    groups = [(int(n), int(p)) for n, p in zip(rng.integers(0, 5, 150), rng.integers(0, 6, 150))]
    case = S.SpanCase(34, rows(rng, groups, 40), groups=groups, kv_heads=2)
    got, err = run(case)
    assert err == 0
    S.check(got, case)


def test_two_groups_on_the_same_pages():
    """A prefix that two groups name."""
    case = S.SpanCase(35, [70, 64, 90, 100], groups=[(2, 3), (2, 3)])
    case.prefix_tables[1] = case.prefix_tables[0]
    case.full[2:, :3] = case.prefix_tables[0, :3]
    got, err = run(case)
    assert err == 0
    S.check(got, case)


def test_one_workspace_for_both_decode_forms():
    """Calls of both forms and of different sizes in turn on one workspace."""
    import test_window_attention_gpu as T
    groups = [(9, 21), (36, 13)]
    shared = S.SpanCase(36, rows(np.random.default_rng(7), groups, 300), groups=groups)
    windows = S.SpanCase(37, [700, 33, 1, 3000, 250, 17, 1600, 0, 16], window=900, sinks=20)
    ws = ops.SpanWorkspace(45, "cuda", max_groups=2)
    for _ in range(3):
        for case, call in ((shared, run), (windows, T.run_decode)):
            got, err = call(case, workspace=ws)
            assert err == 0
            S.check(got, case)
