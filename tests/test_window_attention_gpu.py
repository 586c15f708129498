"""Windowed attention with sinks on the GPU, decode and prefill, against the
64-bit oracle, with NaN in every slot that no query may see and -1 in the table
entries of pages that hold no visible token."""
import numpy as np
import pytest
import torch

import span_cases as S
from gpu_util import dev_bf16, dev_i32, host_bf16
from vllm_b200 import _native as N
from vllm_b200 import ops

pytestmark = pytest.mark.gpu


def run_decode(case, num_ctas=0, out=None, workspace=None, stream=None):
    err = ops.new_error_word("cuda")
    ws = workspace or ops.SpanWorkspace(len(case.lens), "cuda", num_ctas=num_ctas, kv_heads=case.kv_heads)
    got = ops.paged_window_decode_attention(
        dev_bf16(case.q), dev_bf16(case.k_pool), dev_bf16(case.v_pool), case.layer, dev_i32(case.tables),
        dev_i32(case.lens), case.window, ws, sinks=case.sinks, scale=case.scale, out=out, error=err,
        stream=stream)
    torch.cuda.synchronize()
    return host_bf16(got), int(err.item())


def run_prefill(case, out=None, max_q=None):
    err = ops.new_error_word("cuda")
    got = ops.paged_window_prefill_attention(
        dev_bf16(case.q), dev_bf16(case.k_pool), dev_bf16(case.v_pool), case.layer, dev_i32(case.tables),
        dev_i32(case.cu_q), dev_i32(case.q_pos0), int(case.q_counts.max()) if max_q is None else max_q,
        case.window, sinks=case.sinks, scale=case.scale, out=out, error=err)
    torch.cuda.synchronize()
    return host_bf16(got), int(err.item())


EDGE_LENS = [[1], [2], [16], [17], [15, 16, 17, 31, 32, 33], [0, 5, 0, 40, 0], [257, 1, 1000, 64, 0, 129, 700]]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (15, 0), (16, 16), (17, 1), (33, 4), (64, 0),
                                          (100, 17), (128, 33), (500, 100), (5000, 4)])
@pytest.mark.parametrize("lens", EDGE_LENS, ids=str)
def test_decode_edges(lens, window, sinks):
    case = S.SpanCase(11 + window, lens, window=window, sinks=sinks)
    got, err = run_decode(case)
    assert err == 0
    S.check(got, case, f"{lens} window {window} sinks {sinks}")


@pytest.mark.parametrize("kv_heads", [1, 2, 4, 8])
@pytest.mark.parametrize("ctas", [1, 3, 7, 148, 500])
def test_decode_any_heads_and_grid(kv_heads, ctas):
    case = S.SpanCase(20 + kv_heads, [700, 33, 1, 3000, 250, 17, 1600, 0, 16], kv_heads=kv_heads, window=900,
                      sinks=20, num_layers=2, layer=1)
    got, err = run_decode(case, num_ctas=ctas)
    assert err == 0
    S.check(got, case, f"heads {kv_heads} ctas {ctas}")


def test_decode_random_rows_and_one_workspace():
    """One workspace serves calls of any batch, in any order, and a call's bits do not change."""
    rng = np.random.default_rng(5)
    ws = ops.SpanWorkspace(300, "cuda")
    first = None
    for n in (300, 3, 37, 300):
        lens = rng.integers(0, 600, n) if n < 300 else np.random.default_rng(6).integers(0, 600, n)
        case = S.SpanCase(n, lens, window=200, sinks=5)
        got, err = run_decode(case, workspace=ws)
        assert err == 0
        S.check(got, case, f"{n} rows")
        if n == 300:
            assert first is None or np.array_equal(first, got)
            first = got


def test_decode_split_rows_repeat_bit_for_bit():
    case = S.SpanCase(31, [95 * 16, 16, 160 * 16], window=150 * 16, sinks=3, kv_heads=2)
    ref, err = run_decode(case, num_ctas=8)
    assert err == 0
    S.check(ref, case)
    ws = ops.SpanWorkspace(3, "cuda", num_ctas=8, kv_heads=2)
    for _ in range(20):
        got, err = run_decode(case, workspace=ws)
        assert err == 0 and np.array_equal(got, ref)


def test_decode_wide_scores_and_other_scales():
    """Scores of some hundreds: the running maximum has to move, and other scales than 1/8."""
    case = S.SpanCase(40, [300, 77, 1500], window=400, sinks=8, scale=0.3)
    got, err = run_decode(case)
    assert err == 0
    S.check(got, case)


def test_whole_window_equals_plain_decode_attention():
    """A window over the whole row is K2's attention: same tolerance against the same oracle."""
    case = S.SpanCase(50, [900, 40, 2000, 129], window=1 << 30, sinks=0)
    got, err = run_decode(case)
    assert err == 0
    S.check(got, case)


def test_windows_and_sinks_past_32_bits_see_everything():
    case = S.SpanCase(51, [300, 17], window=1 << 30, sinks=0)
    for window, sinks in ((1 << 33, 0), (1, (1 << 32) + 1)):
        case.window, case.sinks = window, sinks
        got, err = run_decode(case)
        assert err == 0
        S.check(got, case)
    prompt = S.SpanCase(52, [70], window=1 << 30, sinks=0, q_counts=[70])
    prompt.window = (1 << 32) + 2
    got, err = run_prefill(prompt)
    assert err == 0
    S.check(got, prompt)


def test_decode_bad_pages_and_lengths_are_reported():
    case = S.SpanCase(60, [300, 60, 45], window=100, sinks=4)
    ok, _ = run_decode(case)
    bad = S.SpanCase(60, [300, 60, 45], window=100, sinks=4)
    bad.tables[0, 15] = bad.num_pages + 5
    got, err = run_decode(bad)
    assert err == N.TVP_DEVERR_BAD_PAGE
    assert np.array_equal(got[1:], ok[1:])
    bad = S.SpanCase(60, [300, 60, 45], window=100, sinks=4)
    bad.lens[2] = -3
    got, err = run_decode(bad)
    assert err == N.TVP_DEVERR_BAD_LENGTH
    assert np.array_equal(got[:2], ok[:2]) and (got[2] == 0).all()


def test_decode_captured_and_replayed_with_new_lengths():
    """A captured call reads the lengths and tables of each replay."""
    big = S.SpanCase(70, [500, 20, 333, 64], window=120, sinks=6)
    small = S.SpanCase(70, [480, 1, 0, 63], window=120, sinks=6)
    q, k, v = dev_bf16(big.q), dev_bf16(big.k_pool), dev_bf16(big.v_pool)
    tables, lens = dev_i32(big.tables), dev_i32(big.lens)
    ws, err, out = ops.SpanWorkspace(4, "cuda"), ops.new_error_word("cuda"), torch.empty_like(q)

    def call():
        ops.paged_window_decode_attention(q, k, v, 0, tables, lens, 120, ws, sinks=6, out=out, error=err)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    for case in (big, small, big):
        q.copy_(dev_bf16(case.q))
        k.view(-1)[:dev_bf16(case.k_pool).numel()].copy_(dev_bf16(case.k_pool).view(-1))
        v.view(-1)[:dev_bf16(case.v_pool).numel()].copy_(dev_bf16(case.v_pool).view(-1))
        tables.fill_(-1)
        tables[:, :case.tables.shape[1]].copy_(dev_i32(case.tables))
        lens.copy_(dev_i32(case.lens))
        graph.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        S.check(host_bf16(out), case)


@pytest.mark.parametrize("kv_heads", [1, 2, 4, 8])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (16, 0), (33, 4), (64, 64), (100, 17), (4000, 4)])
def test_prefill_chunks(kv_heads, window, sinks):
    """Prompts and chunks after cached tokens, odd sizes, a sequence without queries."""
    case = S.SpanCase(80 + window + kv_heads, [1, 33, 200, 150, 64, 700, 16], kv_heads=kv_heads, window=window,
                      sinks=sinks, q_counts=[1, 33, 70, 31, 0, 130, 16])
    got, err = run_prefill(case)
    assert err == 0
    S.check(got, case, f"heads {kv_heads} window {window} sinks {sinks}")


@pytest.mark.parametrize("window", [1, 3, 20, 64])
@pytest.mark.parametrize("sinks", [64, 100, 500, 1 << 30])
def test_prefill_sinks_that_reach_past_the_queries(window, sinks):
    """Sinks beyond a tile's own positions, whose chunks are not visible as a whole."""
    case = S.SpanCase(88, [52, 113, 700, 63], kv_heads=2, window=window, sinks=sinks, q_counts=[3, 40, 300, 1])
    got, err = run_prefill(case)
    assert err == 0
    S.check(got, case, f"window {window} sinks {sinks}")


@pytest.mark.parametrize("sinks", [100, 1 << 30])
def test_decode_sinks_past_the_window(sinks):
    case = S.SpanCase(89, [52, 113, 700, 63], window=1, sinks=sinks)
    got, err = run_decode(case)
    assert err == 0
    S.check(got, case)


@pytest.mark.parametrize("window,sinks", [(200, 4), (513, 0), (129, 130)])
def test_prefill_longer_prompts(window, sinks):
    case = S.SpanCase(90, [1500, 900], kv_heads=2, window=window, sinks=sinks, q_counts=[1500, 77], num_layers=2,
                      layer=1)
    got, err = run_prefill(case)
    assert err == 0
    S.check(got, case)


def test_prefill_of_one_token_each_is_decode():
    """Single queries give what the decode form gives, within both tolerances."""
    lens = [700, 33, 1, 129, 16]
    case = S.SpanCase(91, lens, window=60, sinks=5, q_counts=[1] * 5)
    got, err = run_prefill(case)
    assert err == 0
    S.check(got, case)
    dec, err = run_decode(case)
    assert err == 0
    S.check(dec, case)


def test_prefill_leaves_rows_behind_the_last_sequence():
    case = S.SpanCase(92, [70, 40], kv_heads=2, window=30, sinks=2, q_counts=[70, 9])
    q = np.concatenate([case.q, case.q[:5]])
    out = torch.full((q.shape[0], q.shape[1]), 7.0, dtype=torch.bfloat16, device="cuda")
    keep, case.q = case.q, q
    got, err = run_prefill(case, out=out)
    case.q = keep
    assert err == 0
    S.check(got[:len(keep)], case)
    assert (W_f32(got[len(keep):]) == 7.0).all()


def W_f32(bits):
    import workloads as W
    return W.bf16_to_f32(bits)


def test_prefill_bad_page_and_position():
    case = S.SpanCase(93, [200, 64], kv_heads=2, window=50, sinks=2, q_counts=[30, 64])
    ok, _ = run_prefill(case)
    bad = S.SpanCase(93, [200, 64], kv_heads=2, window=50, sinks=2, q_counts=[30, 64])
    bad.tables[0, 12] = -7
    got, err = run_prefill(bad)
    assert err == N.TVP_DEVERR_BAD_PAGE and np.array_equal(got[30:], ok[30:])
    bad = S.SpanCase(93, [200, 64], kv_heads=2, window=50, sinks=2, q_counts=[30, 64])
    bad.q_pos0[0] = -1
    got, err = run_prefill(bad)
    assert err & N.TVP_DEVERR_BAD_TOKEN and np.array_equal(got[30:], ok[30:])


def test_calls_on_another_stream():
    case = S.SpanCase(94, [300, 20], window=64, sinks=4)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got, err = run_decode(case, stream=side)
    assert err == 0
    S.check(got, case)
