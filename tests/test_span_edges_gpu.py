"""Edges of the windowed and shared-prefix attention on the GPU, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import span_cases as S
import test_shared_prefix_gpu as P
import test_window_attention_gpu as T
from gpu_util import dev_bf16, dev_i32, host_bf16
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


def test_many_groups_captured_and_replayed_with_other_groups():
    """A captured call reads the group rows, prefixes and lengths of each replay, its plan among them."""
    rng = np.random.default_rng(12)
    cases = []
    for seed in (1, 2, 3):
        groups = [(1, int(p)) for p in rng.integers(0, 6, 200)]
        order = rng.permutation(200)
        cases.append(S.SpanCase(400 + seed, P.rows(rng, [groups[i] for i in order], 50),
                                groups=[groups[i] for i in order], kv_heads=1))
    pages, stride = max(c.num_pages for c in cases), max(c.tables.shape[1] for c in cases)
    pstride = max(c.prefix_tables.shape[1] for c in cases)

    def inputs(c):
        def wide(a, shape, fill):
            out = np.full(shape, fill, a.dtype)
            out[tuple(slice(n) for n in a.shape)] = a
            return out
        pool = (1, pages, 16, 64)
        return [dev_bf16(c.q), dev_bf16(wide(c.k_pool, pool, 0x7FC0)), dev_bf16(wide(c.v_pool, pool, 0x7FC0)),
                dev_i32(wide(c.tables, (200, stride), -1)), dev_i32(c.lens),
                dev_i32(wide(c.prefix_tables, (200, pstride), -1)), dev_i32(c.prefix_pages), dev_i32(c.group_rows)]
    args = inputs(cases[0])
    ws, err, out = ops.SpanWorkspace(200, "cuda", kv_heads=1, max_groups=200), ops.new_error_word("cuda"), \
        torch.empty_like(args[0])

    def call():
        ops.paged_shared_prefix_decode_attention(args[0], args[1], args[2], 0, *args[3:], ws, out=out, error=err)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    for case in cases + cases[:1]:
        for to, new in zip(args, inputs(case)):
            to.copy_(new)
        out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        S.check(host_bf16(out), case)


@pytest.mark.parametrize("form", ["decode", "prefill", "shared"])
def test_pages_behind_four_gigabytes(form):
    """The same pages, in a small pool and at the end of one of 4.7 GB (second of two layers)."""
    if form == "shared":
        case = S.SpanCase(71, [100, 64, 300, 17], groups=[(3, 4)])
    else:
        case = S.SpanCase(72, [300, 17, 90], window=70, sinks=5,
                          q_counts=None if form == "decode" else [40, 17, 3])
    pages = 144_000
    pools = []
    for bits in (case.k_pool, case.v_pool):
        pool = torch.empty((2, pages, 16, 512), dtype=torch.bfloat16, device="cuda")
        pool[1, pages - case.num_pages:].copy_(dev_bf16(bits)[0])
        pools.append(pool)
    assert pools[0].numel() * 2 > 1 << 32

    def moved(table):
        return dev_i32(np.where(table < 0, table, table + pages - case.num_pages))
    q, err = dev_bf16(case.q), ops.new_error_word("cuda")
    ws = ops.SpanWorkspace(len(case.lens), "cuda", max_groups=1)
    if form == "decode":
        out = ops.paged_window_decode_attention(q, *pools, 1, moved(case.tables), dev_i32(case.lens), case.window, ws,
                                                sinks=case.sinks, error=err)
    elif form == "prefill":
        out = ops.paged_window_prefill_attention(q, *pools, 1, moved(case.tables), dev_i32(case.cu_q),
                                                 dev_i32(case.q_pos0), 40, case.window, sinks=case.sinks, error=err)
    else:
        out = ops.paged_shared_prefix_decode_attention(
            q, *pools, 1, moved(case.tables), dev_i32(case.lens), moved(case.prefix_tables),
            dev_i32(case.prefix_pages), dev_i32(case.group_rows), ws, error=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    S.check(host_bf16(out), case)
