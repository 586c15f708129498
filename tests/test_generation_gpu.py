"""The windowed and shared-prefix attention and the sampler as a serving loop
uses them: a shared system prompt, ragged prompts behind it, then decode steps
of two layers (one windowed, one over the whole context with the prefix read
once), the LM head and a drawn token, eager and as a replayed graph.  Every
step is checked against 64-bit attention over the pools' own contents and the
definition of the draw over the step's own logits."""
import numpy as np
import pytest
import torch

import span_cases as S
from gpu_util import f32, host_bf16
from sample_oracle import sample_row
from vllm_b200 import ops

pytestmark = pytest.mark.gpu

PREFIX_PAGES, WINDOW, SINKS, VOCAB, DIM = 3, 24, 4, 1008, 2048
PROMPTS = [1, 20, 7, 16, 90]  # own tokens; the last row shares nothing


class Engine:
    """Pools, tables and weights of the loop; every run starts from the same state."""

    def __init__(self):
        g = torch.Generator("cuda").manual_seed(3)
        normal = lambda *s, by=1.0: (torch.randn(*s, generator=g, device="cuda") * by).bfloat16()  # noqa: E731
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        rows = len(PROMPTS)
        self.shared = [1] * (rows - 1) + [0]  # rows behind the prefix
        stride = 10
        perm = torch.randperm(rows * stride + PREFIX_PAGES + 2, generator=g, device="cuda").to(torch.int32)
        self.prefix = perm[:PREFIX_PAGES][None].contiguous()
        self.tables = perm[PREFIX_PAGES:PREFIX_PAGES + rows * stride].view(rows, stride).contiguous()
        self.tables[:rows - 1, :PREFIX_PAGES] = self.prefix
        pool = (2, perm.numel(), 16, 512)
        self.k_pool = torch.full(pool, float("nan"), dtype=torch.bfloat16, device="cuda")
        self.v_pool = self.k_pool.clone()
        self.lens = i32([PREFIX_PAGES * 16 * s + n for s, n in zip(self.shared, PROMPTS)])
        self.prefix_pages, self.group_rows = i32([PREFIX_PAGES]), i32([0, rows - 1])
        self.embed = normal(VOCAB, DIM)
        self.w = [[normal(n, DIM, by=DIM ** -0.5) for n in (2048, 512, 512)] for _ in range(2)]
        self.w_o, self.w_head = normal(DIM, DIM, by=DIM ** -0.5), normal(VOCAB, DIM, by=0.2)
        self.temperature = torch.tensor([1.0, 0.7, 0.0, 1.3, 0.9], device="cuda")
        self.top_k, self.top_p = i32([0, 50, 0, 400, 7]), torch.tensor([1.0, 0.9, 1.0, 0.8, 0.95], device="cuda")
        self.tokens, self.uniforms = i32([5, 900, 33, 1, 77]), torch.zeros(rows, device="cuda")
        self.err = ops.new_error_word("cuda")
        self.ws = ops.SpanWorkspace(rows, "cuda", max_groups=1)
        self.prefill(normal)

    def prefill(self, normal):
        """Appends the prefix once, then every row's prompt; returns nothing, checks layer 0's attention."""
        n = PREFIX_PAGES * 16
        for layer in range(2):
            pos = torch.arange(n, dtype=torch.int32, device="cuda")
            ops.rope_append(self.k_pool, self.v_pool, layer, self.prefix, pos, normal(n, 512), normal(n, 512),
                            token_seq=torch.zeros_like(pos), error=self.err)
        start = [PREFIX_PAGES * 16 * s for s in self.shared]
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, PROMPTS)]).to(torch.int32).cuda()
        seq = torch.repeat_interleave(torch.arange(len(PROMPTS)), torch.tensor(PROMPTS)).to(torch.int32).cuda()
        cu = torch.tensor(np.cumsum([0] + PROMPTS), dtype=torch.int32, device="cuda")
        for layer in range(2):
            q = normal(pos.numel(), 2048)
            ops.rope_append(self.k_pool, self.v_pool, layer, self.tables, pos, normal(pos.numel(), 512),
                            normal(pos.numel(), 512), q=q, token_seq=seq, error=self.err)
            window, sinks = (WINDOW, SINKS) if layer == 0 else (1 << 20, 0)
            out = ops.paged_window_prefill_attention(
                q, self.k_pool, self.v_pool, layer, self.tables, cu, torch.tensor(start, dtype=torch.int32).cuda(),
                max(PROMPTS), window, sinks=sinks, error=self.err)
            torch.cuda.synchronize()
            assert int(self.err.item()) == 0
            self.check_attention(layer, q, out, seq.tolist(), pos.tolist(), window, sinks)

    def step(self):
        """One decode step of every row on the current stream: no host work depends on the device."""
        self.lens.add_(1)
        pos = self.lens - 1
        x, seen = self.embed[self.tokens.long()], []
        for layer in range(2):
            q, k, v = ops.decode_projections(x, self.w[layer])
            ops.rope_append(self.k_pool, self.v_pool, layer, self.tables, pos, k, v, q=q, error=self.err)
            if layer == 0:
                attn = ops.paged_window_decode_attention(q, self.k_pool, self.v_pool, layer, self.tables, self.lens,
                                                         WINDOW, self.ws, sinks=SINKS, error=self.err)
            else:
                attn = ops.paged_shared_prefix_decode_attention(
                    q, self.k_pool, self.v_pool, layer, self.tables, self.lens, self.prefix, self.prefix_pages,
                    self.group_rows, self.ws, error=self.err)
            seen.append((q, attn))
            x = x + ops.decode_projections(attn, [self.w_o])[0]
        logits = ops.decode_projections(x, [self.w_head], epilogue="f32")[0]
        ops.sample_tokens(logits, self.uniforms, self.temperature, self.top_k, self.top_p, out=self.tokens)
        return seen, logits

    def check_attention(self, layer, q, out, rows, positions, window, sinks):
        q, out = (f32(host_bf16(t)).astype(np.float64) for t in (q, out))
        k, v = (f32(host_bf16(t[layer])).astype(np.float64) for t in (self.k_pool, self.v_pool))
        tables = self.tables.cpu().numpy()
        for i, (row, pos) in enumerate(zip(rows, positions)):
            at = S.visible(pos, window, sinks)
            phys = tables[row, at // 16]
            for h in range(8):
                cols = slice(h * 256, (h + 1) * 256)
                o, a = S.attend(q[i, cols].reshape(4, 64), k[phys, at % 16, h * 64:h * 64 + 64],
                                v[phys, at % 16, h * 64:h * 64 + 64], 0.125)
                tol = 2.0 ** -8 * (a + 2 * np.abs(o)) + 2.0 ** -13 * a
                assert (np.abs(out[i, cols].reshape(4, 64) - o) <= tol).all(), (layer, i, h)

    def check_step(self, seen, logits):
        assert int(self.err.item()) == 0
        rows, positions = range(len(PROMPTS)), (self.lens - 1).tolist()
        for layer, (q, attn) in enumerate(seen):
            self.check_attention(layer, q, attn, rows, positions, *((WINDOW, SINKS) if layer == 0 else (1 << 20, 0)))
        x, u, got = logits.cpu().numpy(), self.uniforms.cpu().numpy(), self.tokens.tolist()
        for r in rows:
            want, near = sample_row(x[r], u[r], float(self.temperature[r]), int(self.top_k[r]),
                                    np.float32(self.top_p[r].item()))
            assert near > VOCAB * 2.0 ** -43 and got[r] == want, (r, near, got[r], want)


def draws(step):
    return torch.from_numpy(np.random.default_rng(100 + step).random(len(PROMPTS), dtype=np.float32))


def test_decode_loop_eager_and_captured():
    eager, tokens = Engine(), []
    for i in range(20):  # rows pass a page's end on the way
        eager.uniforms.copy_(draws(i))
        result = eager.step()
        torch.cuda.synchronize()
        eager.check_step(*result)
        tokens.append(eager.tokens.tolist())
    assert len({t for row in tokens for t in row}) > 10

    engine, side = Engine(), torch.cuda.Stream()
    state = [engine.lens.clone(), engine.tokens.clone()]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        engine.step()  # warms up; the appended slot is written again by the replay
    side.synchronize()
    engine.lens.copy_(state[0])
    engine.tokens.copy_(state[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        result = engine.step()
    for i in range(20):
        engine.uniforms.copy_(draws(i))
        graph.replay()
        torch.cuda.synchronize()
        assert engine.tokens.tolist() == tokens[i], i
    engine.check_step(*result)


def test_two_loops_at_once():
    """Two engines with a workspace each, on a stream each, step at the same time."""
    one, two = Engine(), Engine()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    two.tokens.add_(7)
    alone = []
    for engine in (Engine(), Engine()):
        if alone:
            engine.tokens.add_(7)
        out = []
        for i in range(8):
            engine.uniforms.copy_(draws(i))
            engine.step()
            out.append(engine.tokens.clone())
        alone.append(torch.stack(out))
    uniforms = torch.stack([draws(i) for i in range(8)]).cuda()
    torch.cuda.synchronize()
    out = [[], []]
    for i in range(8):
        for e, (engine, stream) in enumerate(zip((one, two), streams)):
            with torch.cuda.stream(stream):
                engine.uniforms.copy_(uniforms[i])
                engine.step()
                out[e].append(engine.tokens.clone())
    torch.cuda.synchronize()
    for e, engine in enumerate((one, two)):
        assert int(engine.err.item()) == 0
        assert torch.equal(torch.stack(out[e]), alone[e])
