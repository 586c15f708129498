"""The decode step's further operators, in plain torch and through the framework:
windowed paged attention with sinks (decode and prefill), decode attention of a
batch that shares a prefix, and token sampling.  Each case is one operator at
one size; `run` makes one pass of it."""
import math

import numpy as np
import torch

own = False

PAGE, DIM, GROUP = 16, 64, 4
SCALE = 0.125


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def listed():
    return [
        # One request near the reference engine's 1024-token context, a short window: launch latency.
        {"name": "window_decode_1x1023", "op": "window_decode", "rows": 1, "len_lo": 1023, "len_hi": 1023,
         "window": 256, "sinks": 4, "kv_heads": 8},
        # The decode sweep's 256 ragged rows of 512 to 8192 tokens, four first tokens kept.
        {"name": "window_decode_256x8192", "op": "window_decode", "rows": 256, "len_lo": 512, "len_hi": 8192,
         "window": 2048, "sinks": 4, "kv_heads": 8},
        # The long-context rows on one GPU of a KV-head-sharded deployment (one head of the eight).
        {"name": "window_decode_16x32768_1head", "op": "window_decode", "rows": 16, "len_lo": 32768, "len_hi": 32768,
         "window": 16384, "sinks": 100, "kv_heads": 1},
        # The four 256-token prompts of the append workload, a window shorter than the prompt.
        {"name": "window_prefill_4x256", "op": "window_prefill", "seqs": 4, "q_lo": 256, "q_hi": 256,
         "past_hi": 0, "window": 64, "sinks": 4, "kv_heads": 8},
        # One long prompt.
        {"name": "window_prefill_1x8192", "op": "window_prefill", "seqs": 1, "q_lo": 8192, "q_hi": 8192,
         "past_hi": 0, "window": 2048, "sinks": 4, "kv_heads": 8},
        # Chunked prefill: ragged chunks after up to 4000 cached tokens, two KV heads held.
        {"name": "window_prefill_6x1500_chunks", "op": "window_prefill", "seqs": 6, "q_lo": 1, "q_hi": 1500,
         "past_hi": 4000, "window": 1000, "sinks": 17, "kv_heads": 2},
        # The scheduler's four slots behind a short system prompt.
        {"name": "shared_prefix_4x512", "op": "shared_prefix", "groups": 1, "rows": 4, "prefix_pages": 32,
         "own_hi": 128, "kv_heads": 8},
        # Three tenants with a system prompt each, ragged rows.
        {"name": "shared_prefix_3x37x2048", "op": "shared_prefix", "groups": 3, "rows": 37, "prefix_pages": 128,
         "own_hi": 700, "kv_heads": 8},
        # 256 rows that share one long document.
        {"name": "shared_prefix_256x8192", "op": "shared_prefix", "groups": 1, "rows": 256, "prefix_pages": 512,
         "own_hi": 1024, "kv_heads": 8},
        # One request's logits, the usual chat settings.
        {"name": "sample_1x128256", "op": "sample", "rows": 1, "vocab": 128256, "k_hi": 50, "p_lo": 0.9},
        # A mixed batch of an odd vocabulary.
        {"name": "sample_33x50257", "op": "sample", "rows": 33, "vocab": 50257, "k_hi": 1000, "p_lo": 0.5},
        # 256 rows, each with settings of its own.
        {"name": "sample_256x128256", "op": "sample", "rows": 256, "vocab": 128256, "k_hi": 200, "p_lo": 0.7},
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["window_decode", "window_prefill", "shared_prefix", "sample"])
    if op == "sample":
        rows = _log_int(rng, 1, 256)
        return {"op": op, "rows": rows, "vocab": _log_int(rng, 1000, 128256), "k_hi": _log_int(rng, 1, 2000),
                "p_lo": round(rng.uniform(0.1, 0.99), 3)}
    heads = rng.choice([8, 8, 4, 2, 1])
    if op == "window_decode":
        rows = _log_int(rng, 1, 256)
        hi = _log_int(rng, 1, 32768 if rows <= 16 else 8192)
        return {"op": op, "rows": rows, "len_lo": max(1, hi // rng.choice([1, 2, 16])), "len_hi": hi,
                "window": _log_int(rng, 1, 4096 if rows <= 16 else 2048), "sinks": rng.choice([0, 1, 4, 16, 33, 100]),
                "kv_heads": heads}
    if op == "window_prefill":
        seqs = _log_int(rng, 1, 8)
        past = rng.choice([0, 0, _log_int(rng, 1, 4000 // seqs)])
        hi = _log_int(rng, 1, 8192 // seqs - past)
        return {"op": op, "seqs": seqs, "q_lo": max(1, hi // rng.choice([1, 3, 50])), "q_hi": hi, "past_hi": past,
                "window": _log_int(rng, 1, 2048), "sinks": rng.choice([0, 1, 4, 16, 33, 100]), "kv_heads": heads}
    groups = rng.choice([1, 1, 2, 3, 5])
    return {"op": op, "groups": groups, "rows": _log_int(rng, 1, 256 // groups),
            "prefix_pages": _log_int(rng, 1, 512), "own_hi": _log_int(rng, 1, 1024), "kv_heads": heads}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _spread(case):
    """Query counts of a prefill case: from q_lo to q_hi, in an order that the seed gives."""
    return np.linspace(case["q_lo"], case["q_hi"], case["seqs"]).astype(np.int64)


def _lengths(case, seed):
    """Host-side sizes of a case: they shape the inputs and the count of work."""
    r = np.random.default_rng(seed)
    if case["op"] == "window_decode":
        return {"lens": r.integers(case["len_lo"], case["len_hi"] + 1, case["rows"])}
    if case["op"] == "window_prefill":
        past = r.integers(0, case["past_hi"] + 1, case["seqs"])
        q = r.permutation(_spread(case))
        return {"past": past, "q": q, "lens": past + q}
    if case["op"] == "shared_prefix":
        n = case["groups"] * case["rows"]
        # each group's prefix is a little shorter or longer than the named one
        pages = np.maximum(1, case["prefix_pages"] - np.arange(case["groups"]) * (case["prefix_pages"] // 7))
        tail = r.integers(1, case["own_hi"] + 1, n)
        return {"pages": pages, "lens": np.repeat(pages, case["rows"]) * PAGE + tail}
    return {}


def _normal(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16)


def _device(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed + 1)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a broad body of logits with a few tokens standing out, as a language model's
        logits = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.5
        peaks = torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda")
        logits.scatter_add_(1, peaks, 4.0 + 8.0 * torch.rand((rows, 24), generator=gen, device="cuda"))
        # every row with settings of its own, some without one filter or the other
        temp = r.choice([0.2, 0.7, 1.0, 1.3], rows).astype(np.float32)
        top_k = np.where(r.random(rows) < 0.3, 0, r.integers(1, case["k_hi"] + 1, rows)).astype(np.int32)
        top_p = np.where(r.random(rows) < 0.3, 1.0, r.uniform(case["p_lo"], 1.0, rows)).astype(np.float32)
        min_p = np.where(r.random(rows) < 0.5, 0.0, r.uniform(0.0, 0.1, rows)).astype(np.float32)
        return {"case": case, "logits": logits, "uniforms": torch.rand(rows, generator=gen, device="cuda"),
                "temperature": torch.from_numpy(temp).cuda(), "top_k": torch.from_numpy(top_k).cuda(),
                "top_p": torch.from_numpy(top_p).cuda(), "min_p": torch.from_numpy(min_p).cuda()}
    size = _lengths(case, seed)
    lens, heads = size["lens"], case["kv_heads"]
    need = -(-lens // PAGE)
    stride = int(need.max())
    shared = np.zeros(len(lens), np.int64)
    if case["op"] == "shared_prefix":
        shared = np.repeat(size["pages"], case["rows"])
        total = int((need - shared).sum() + size["pages"].sum())
    else:
        total = int(need.sum())
    pages = r.permutation(total + 3).astype(np.int32)
    tables = np.full((len(lens), stride), -1, np.int32)
    used = 0
    state = {"case": case}
    if case["op"] == "shared_prefix":
        prefix = np.full((case["groups"], int(size["pages"].max())), -1, np.int32)
        for g, n in enumerate(size["pages"]):
            prefix[g, :n] = pages[used:used + n]
            tables[g * case["rows"]:(g + 1) * case["rows"], :n] = prefix[g, :n]
            used += n
        state |= {"prefix_tables": _device(prefix), "prefix_pages": _device(size["pages"]),
                  "group_rows": _device(np.arange(case["groups"] + 1) * case["rows"])}
    for b in range(len(lens)):
        n = int(need[b] - shared[b])
        tables[b, shared[b]:need[b]] = pages[used:used + n]
        used += n
    tokens = len(lens)
    if case["op"] == "window_prefill":
        tokens = int(size["q"].sum())
        state |= {"cu_q": _device(np.concatenate([[0], np.cumsum(size["q"])])), "q_pos0": _device(size["past"]),
                  "max_q": int(size["q"].max())}
    return state | {"k_pool": _normal((1, total + 3, PAGE, heads * DIM), gen),
                    "v_pool": _normal((1, total + 3, PAGE, heads * DIM), gen),
                    "q": _normal((tokens, heads * GROUP * DIM), gen),
                    "tables": _device(tables), "lens": _device(lens), "max_len": int(lens.max())}


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _framework(op, state)
    if op == "sample":
        return _plain_sample(state)
    if op == "window_prefill":
        return _plain_prefill(state)
    return _plain_decode(state)


def _framework(op, s):
    from vllm_b200 import ops
    case = s["case"]
    if op == "sample":
        return ops.sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                 top_p=s["top_p"], min_p=s["min_p"])
    if op == "window_prefill":
        return ops.paged_window_prefill_attention(s["q"], s["k_pool"], s["v_pool"], 0, s["tables"], s["cu_q"],
                                                  s["q_pos0"], s["max_q"], case["window"], sinks=case["sinks"],
                                                  scale=SCALE)
    if "workspace" not in s:  # a serving loop keeps it
        s["workspace"] = ops.SpanWorkspace(s["lens"].numel(), s["q"].device, kv_heads=case["kv_heads"],
                                           max_groups=case.get("groups", 0))
    if op == "window_decode":
        return ops.paged_window_decode_attention(s["q"], s["k_pool"], s["v_pool"], 0, s["tables"], s["lens"],
                                                 case["window"], s["workspace"], sinks=case["sinks"], scale=SCALE)
    return ops.paged_shared_prefix_decode_attention(s["q"], s["k_pool"], s["v_pool"], 0, s["tables"], s["lens"],
                                                    s["prefix_tables"], s["prefix_pages"], s["group_rows"],
                                                    s["workspace"], scale=SCALE)


def _gather(pool, tables, pos):
    """Rows of one layer's pool at token positions `pos` [B, M], in 32 bits: [B, KV heads, M, 64]."""
    page = tables.gather(1, (pos // PAGE)).long().clamp(min=0)
    rows = pool[0].float()[page, pos % PAGE]
    return rows.reshape(*pos.shape, -1, DIM).transpose(1, 2)


def _attend(q, k, v, seen):
    """q [B, G, R, 64] against k, v [B, G, M, 64] where seen [B, 1, R or 1, M]."""
    score = (q @ k.transpose(-1, -2)) * SCALE
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    return (p @ v) / p.sum(-1, keepdim=True)


def _plain_decode(s):
    case, lens = s["case"], s["lens"].long()
    rows, heads = lens.numel(), case["kv_heads"]
    # the positions a row sees: its first ones, then its last ones
    sinks = case.get("sinks", 0)
    window = case.get("window", s["max_len"])
    first = (lens - window).clamp(min=sinks)
    at = torch.arange(min(sinks + window, s["max_len"]), device=lens.device)[None]
    pos = torch.where(at < sinks, at, first[:, None] + at - sinks)
    seen = pos < lens[:, None]
    pos = torch.where(seen, pos, torch.zeros_like(pos))
    k, v = _gather(s["k_pool"], s["tables"], pos), _gather(s["v_pool"], s["tables"], pos)
    q = s["q"].float().reshape(rows, heads, GROUP, DIM)
    return _attend(q, k, v, seen[:, None, None]).reshape(rows, -1).to(torch.bfloat16)


def _plain_prefill(s):
    case = s["case"]
    start, pos0, heads = s["cu_q"].long(), s["q_pos0"].long(), case["kv_heads"]
    at = torch.arange(s["max_q"], device=start.device)[None]
    real = at < (start[1:] - start[:-1])[:, None]  # [S, Q]
    token = torch.where(real, start[:-1, None] + at, torch.zeros_like(at))
    q = s["q"].float()[token].reshape(*token.shape, heads, GROUP, DIM)
    qpos = (pos0[:, None] + at)[:, :, None]
    key = torch.arange(s["max_len"], device=start.device)[None, None]
    seen = (key <= qpos) & ((key > qpos - case["window"]) | (key < case["sinks"]))  # [S, Q, K]
    pos = key[0].expand(pos0.numel(), -1)
    k, v = _gather(s["k_pool"], s["tables"], pos), _gather(s["v_pool"], s["tables"], pos)
    # rows of the product: (token, head of the group)
    q = q.permute(0, 2, 1, 3, 4).reshape(pos0.numel(), heads, -1, DIM)
    out = _attend(q, k, v, seen.repeat_interleave(GROUP, 1)[:, None])
    out = out.reshape(pos0.numel(), heads, s["max_q"], GROUP * DIM).transpose(1, 2)
    return out.reshape(pos0.numel(), s["max_q"], -1)[real].to(torch.bfloat16)


def _plain_sample(s):
    # 64 bits: a token is decided by a running sum next to a border
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(1, keepdim=True)
    weight = torch.exp((x - top) / s["temperature"].double()[:, None])
    order = torch.argsort(x, dim=1, descending=True, stable=True)
    w = weight.gather(1, order)
    rank = torch.arange(x.shape[1], device=x.device)[None]
    k = s["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    before = w.cumsum(1) - w
    p = s["top_p"].double()[:, None]
    kept = (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0)
    kept &= w >= s["min_p"].double()[:, None]
    w = torch.where(kept, w, torch.zeros_like(w))
    run_sum = torch.zeros_like(w).scatter_(1, order, w).cumsum(1)
    point = s["uniforms"].double()[:, None] * run_sum[:, -1:]
    return (run_sum <= point).sum(1).to(torch.int32)


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        x = s["logits"].cpu().numpy().astype(np.float64)
        u, temp, top_p, min_p = (s[n].cpu().numpy().astype(np.float64)
                                 for n in ("uniforms", "temperature", "top_p", "min_p"))
        top_k, tokens = s["top_k"].cpu().numpy(), []
        for r, row in enumerate(x):
            fall = np.lexsort((np.arange(row.size), -row))  # falling, ties by index
            if top_k[r] > 0:
                fall = fall[:top_k[r]]
            mass = np.exp((row[fall] - row[fall[0]]) / temp[r])
            if top_p[r] < 1:
                fall = fall[:1 + int(np.searchsorted(np.cumsum(mass), top_p[r] * mass.sum(), "left"))]
                mass = mass[:fall.size]
            fall, mass = fall[mass >= min_p[r]], mass[mass >= min_p[r]]
            by_index = np.argsort(fall)
            total = np.cumsum(mass[by_index])
            tokens.append(int(fall[by_index[np.searchsorted(total, u[r] * total[-1], "right")]]))
        return torch.tensor(tokens, dtype=torch.int32)
    lens = s["lens"].tolist()
    kp, vp = s["k_pool"][0], s["v_pool"][0]
    heads = case["kv_heads"]
    q_all = s["q"].double().reshape(-1, heads, GROUP, DIM)
    if case["op"] == "window_prefill":
        starts, pos0 = s["cu_q"].tolist(), s["q_pos0"].tolist()
    else:
        starts, pos0 = list(range(len(lens) + 1)), [n - 1 for n in lens]
    out = torch.empty_like(q_all)
    for b, n in enumerate(lens):
        pages = s["tables"][b, :-(-n // PAGE)].long()
        k = kp[pages].reshape(-1, heads, DIM)[:n].double()
        v = vp[pages].reshape(-1, heads, DIM)[:n].double()
        key = torch.arange(n, device=k.device)
        for t0 in range(starts[b], starts[b + 1], 256):
            t1 = min(t0 + 256, starts[b + 1])
            p = torch.arange(t0, t1, device=k.device)[:, None] - starts[b] + pos0[b]
            hidden = key > p
            if "window" in case:
                hidden |= (key <= p - case["window"]) & (key >= case["sinks"])
            score = torch.einsum("tghd,kgd->ghtk", q_all[t0:t1], k) / math.sqrt(DIM)
            prob = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[t0:t1] = torch.einsum("ghtk,kgd->tghd", prob, v)
    return out.reshape(s["q"].shape)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # an exponential (taken as one operation), a comparison and a sum for each logit
        return {"bytes": 4 * n + 24 * case["rows"], "flops": 3 * n}
    # sizes of the mean case: every seed draws lengths of its own
    heads, kv = case["kv_heads"], case["kv_heads"] * DIM * 2 * 2
    row = 2 * 2 * GROUP * heads * DIM  # q and out
    pair = 4 * DIM * GROUP * heads     # q.k and p.v of one query token and key
    if case["op"] == "window_decode":
        mean = np.arange(case["len_lo"], case["len_hi"] + 1)
        seen = float(np.minimum(mean, np.minimum(case["sinks"], np.maximum(mean - case["window"], 0))
                                + np.minimum(mean, case["window"])).mean()) * case["rows"]
        return {"bytes": seen * kv + case["rows"] * row, "flops": seen * pair}
    if case["op"] == "window_prefill":
        past, total = case["past_hi"] // 2, {"bytes": 0, "flops": 0.0}
        for q in _spread(case):
            p = past + np.arange(q)
            seen = np.minimum(p + 1, case["window"]) + np.minimum(case["sinks"], np.maximum(p + 1 - case["window"], 0))
            keys = min(past + q, q + case["window"] - 1 + case["sinks"])
            total["bytes"] += int(keys * kv + q * row)
            total["flops"] += float(seen.sum()) * pair
        return total
    pages = sum(max(1, case["prefix_pages"] - g * (case["prefix_pages"] // 7)) for g in range(case["groups"]))
    rows = case["groups"] * case["rows"]
    tail = rows * (case["own_hi"] + 1) / 2
    return {"bytes": (pages * PAGE + tail) * kv + rows * row, "flops": (case["rows"] * pages * PAGE + tail) * pair}
