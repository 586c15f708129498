"""What the windowed and shared-prefix attention and the sampler refuse, on the
host, before any CUDA call (fake, never dereferenced pointers; no GPU needed)."""
import ctypes

import pytest
import torch

from vllm_b200 import _native as N
from vllm_b200 import ops

FAKE, ODD = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10008)
INVALID, UNSUPPORTED, WORKSPACE = N.TVP_ERR_INVALID_ARGUMENT, N.TVP_ERR_UNSUPPORTED, N.TVP_ERR_WORKSPACE

POOLS = [("q", FAKE), ("k", FAKE), ("v", FAKE), ("pages", 8), ("layers", 16), ("layer", 0), ("kvh", 8), ("qh", 32),
         ("tables", FAKE), ("stride", 4)]
END = [("scale", 0.125), ("ctas", 148), ("ws", FAKE), ("wsb", 1 << 30), ("out", FAKE), ("err", None), ("stream", None)]
WINDOW = POOLS + [("lens", FAKE), ("batch", 2), ("window", 64), ("sinks", 4)] + END
SHARED = POOLS + [("lens", FAKE), ("batch", 2), ("ptables", FAKE), ("pstride", 4), ("ppages", FAKE), ("rows", FAKE),
                  ("groups", 1)] + END
PREFILL = POOLS + [("cu", FAKE), ("pos0", FAKE), ("seqs", 2), ("maxq", 7), ("window", 64), ("sinks", 4),
                   ("scale", 0.125), ("out", FAKE), ("err", None), ("stream", None)]
SAMPLE = [("logits", FAKE), ("rows", 2), ("vocab", 100), ("row_stride", 100), ("u", FAKE), ("t", None), ("k", None),
          ("p", None), ("m", None), ("tokens", FAKE), ("stream", None)]

COMMON = [({"q": None}, INVALID), ({"k": None}, INVALID), ({"v": None}, INVALID), ({"out": None}, INVALID),
          ({"tables": None}, INVALID), ({"pages": 0}, INVALID), ({"layer": 16}, INVALID), ({"layer": -1}, INVALID),
          ({"stride": 0}, INVALID), ({"scale": float("nan")}, INVALID), ({"scale": float("inf")}, INVALID),
          ({"kvh": 3, "qh": 12}, UNSUPPORTED), ({"kvh": 16, "qh": 64}, UNSUPPORTED), ({"qh": 16}, UNSUPPORTED),
          ({"pages": 1 << 24}, UNSUPPORTED), ({"k": ODD}, INVALID), ({"out": ODD}, INVALID),
          ({"stride": 1 << 27}, UNSUPPORTED)]
ROWS = [({"lens": None}, INVALID), ({"batch": 0}, INVALID), ({"batch": -1}, INVALID), ({"ctas": -1}, INVALID),
        ({"ctas": 1025}, INVALID), ({"ws": None}, WORKSPACE), ({"wsb": 1 << 10}, WORKSPACE), ({"ws": ODD}, WORKSPACE)]
WIN = [({"window": 0}, INVALID), ({"window": -5}, INVALID), ({"sinks": -1}, INVALID)]


def refused(fn, args, cases):
    for over, code in cases:
        a = dict(args)
        assert set(over) <= set(a)
        a.update(over)
        assert fn(*a.values()) == code, over


def test_window_decode_refuses(native):
    refused(native.tvp_paged_window_decode_attention, WINDOW, COMMON + ROWS + WIN)


def test_shared_prefix_refuses(native):
    refused(native.tvp_paged_shared_prefix_decode_attention, SHARED, COMMON + ROWS + [
        ({"groups": -1}, INVALID), ({"groups": 65536}, INVALID), ({"ptables": None}, INVALID),
        ({"ppages": None}, INVALID), ({"rows": None}, INVALID), ({"pstride": 0}, INVALID),
        ({"pstride": 1 << 27}, UNSUPPORTED), ({"q": ODD}, INVALID)])


def test_window_prefill_refuses(native):
    refused(native.tvp_paged_window_prefill_attention, PREFILL, COMMON + WIN + [
        ({"cu": None}, INVALID), ({"pos0": None}, INVALID), ({"seqs": 0}, INVALID), ({"seqs": 65536}, INVALID),
        ({"maxq": -1}, INVALID), ({"maxq": 65535 * 32 + 1}, UNSUPPORTED), ({"q": ODD}, INVALID),
        ({"maxq": 0}, N.TVP_OK)])  # nothing to attend: no launch


def test_sampler_refuses(native):
    refused(native.tvp_sample_tokens, SAMPLE, [
        ({"logits": None}, INVALID), ({"u": None}, INVALID), ({"tokens": None}, INVALID), ({"rows": 0}, INVALID),
        ({"vocab": 0}, INVALID), ({"row_stride": 99}, INVALID), ({"logits": ctypes.c_void_p(0x10002)}, INVALID),
        ({"rows": 65536}, UNSUPPORTED),
        ({"vocab": 327681, "row_stride": 327681}, UNSUPPORTED)])


def test_span_workspace_bytes(native):
    f = native.tvp_span_workspace_bytes
    assert f(0, 0, 8, 148) == f(4, -1, 8, 148) == f(4, 0, 3, 148) == f(4, 0, 8, 1025) == f(4, 0, 8, -1) == 0
    assert 0 < f(4, 0, 1, 148) < f(4, 0, 8, 148) < f(4, 1, 8, 148) <= f(400, 1, 8, 148) <= f(100000, 1, 8, 148)
    assert f(4, 1, 8, 148) % 256 == 0
    assert f(4, 0, 8, 148) == f(256, 0, 8, 148)  # the split rows' places go by the grid


def test_python_layer_refuses_host_tensors_and_other_shapes():
    bf, i32 = torch.bfloat16, torch.int32
    pool, q = torch.zeros(1, 2, 16, 512, dtype=bf), torch.zeros(1, 2048, dtype=bf)
    one = torch.zeros(1, dtype=i32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_window_decode_attention(q, pool, pool, 0, one[None], one, 4, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_shared_prefix_decode_attention(q, pool, pool, 0, one[None], one, one[None], one, one, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_window_prefill_attention(q, pool, pool, 0, one[None], one, one, 1, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_tokens(torch.zeros(1, 5), torch.zeros(1))


@pytest.mark.gpu
def test_python_layer_refuses_on_the_gpu():
    bf, i32 = torch.bfloat16, torch.int32
    pool = torch.zeros(1, 4, 16, 512, dtype=bf, device="cuda")
    q, lens = torch.zeros(2, 2048, dtype=bf, device="cuda"), torch.ones(2, dtype=i32, device="cuda")
    tables = torch.zeros(2, 1, dtype=i32, device="cuda")
    ws = ops.SpanWorkspace(2, "cuda", max_groups=1)
    window = lambda **k: ops.paged_window_decode_attention(**{**dict(  # noqa: E731
        q=q, k_pool=pool, v_pool=pool, layer=0, block_tables=tables, seq_lens=lens, window=4, workspace=ws), **k})
    window()
    for bad in ({"window": 0}, {"sinks": -1}, {"layer": 1}, {"q": q[:1]}, {"q": q.float()}, {"block_tables": tables[:1]},
                {"seq_lens": lens.long()}, {"workspace": None}, {"workspace": ops.SpanWorkspace(1, "cuda")},
                {"workspace": ops.SpanWorkspace(2, "cuda", kv_heads=4)}, {"out": q[:1]}, {"error": lens.long()},
                {"v_pool": pool[:, :2]}):
        with pytest.raises(ValueError):
            window(**bad)
    pages, rows = torch.ones(1, dtype=i32, device="cuda"), torch.tensor([0, 2], dtype=i32, device="cuda")
    for bad in ({"prefix_pages": pages.repeat(2)}, {"group_rows": rows[:1]}, {"prefix_tables": tables[:0]},
                {"workspace": ops.SpanWorkspace(2, "cuda")}):
        with pytest.raises(ValueError):
            ops.paged_shared_prefix_decode_attention(**{**dict(
                q=q, k_pool=pool, v_pool=pool, layer=0, block_tables=tables, seq_lens=lens, prefix_tables=tables,
                prefix_pages=pages, group_rows=rows, workspace=ws), **bad})
    x, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for bad in ({"logits": x.t()}, {"logits": x.half()}, {"uniforms": u[:1]}, {"temperature": u.double()},
                {"top_k": u}, {"top_p": u[:1]}, {"out": torch.zeros(1, dtype=i32, device="cuda")}):
        with pytest.raises(ValueError):
            ops.sample_tokens(**{**dict(logits=x, uniforms=u), **bad})
