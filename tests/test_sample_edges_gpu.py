"""Edges of the token sampler on the GPU, in each of its forms (16, 8, 4 or 2 CTAs
a row), against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from sample_oracle import sample_row
from vllm_b200 import ops

pytestmark = pytest.mark.gpu

UNSET = -77


def draw(x, u, **settings):
    """Tokens of rows of FP32 logits; `out` holds UNSET before the call."""
    dev = {k: torch.tensor(np.asarray(v, np.int32 if k == "top_k" else np.float32)).cuda()
           for k, v in settings.items()}
    out = torch.full((len(x),), UNSET, dtype=torch.int32, device="cuda")
    ops.sample_tokens(torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda(),
                      torch.tensor(np.asarray(u, np.float32)).cuda(), out=out, **dev)
    return out.cpu().numpy()


@pytest.mark.parametrize("rows", [1, 5, 63, 64, 191, 192, 500])
@pytest.mark.parametrize("vocab", [1, 2, 5, 40])
def test_rows_shorter_than_their_cluster(rows, vocab):
    """CTAs with few logits or none reach the exchange with the others at once."""
    rng = np.random.default_rng(100 * rows + vocab)
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    xs = torch.from_numpy(x).cuda()
    for k in (0, 3):
        u = rng.random(rows).astype(np.float32)
        want = [sample_row(x[r], u[r], top_k=k) for r in range(rows)]
        assert all(near > vocab * 2.0 ** -43 or near == 0 for _, near in want)
        us, ks = torch.from_numpy(u).cuda(), torch.full((rows,), k, dtype=torch.int32, device="cuda")
        got = [ops.sample_tokens(xs, us, top_k=ks) for _ in range(20)]
        for g in got:
            assert g.tolist() == [w for w, _ in want]


@pytest.mark.parametrize("rows", [1, 8, 70, 200])
@pytest.mark.parametrize("top", [1e7, 20.0, -3.5])
@pytest.mark.parametrize("step", [0.04, 0.045, 0.075, 0.2])
def test_temperatures_below_the_tops_last_place(rows, top, step):
    """Temperature `step` of the top's last place: every logit but the top is more than
    20 of these steps lower and has no weight, whatever the subtraction that finds
    the first such logit rounds to; so every uniform takes the top, first or last of its row."""
    vocab = 70001
    rng = np.random.default_rng(rows)
    top = np.float32(top)
    x = (top - np.float32(4) * np.spacing(np.abs(top)) * rng.integers(20, 1 << 18, (rows, vocab))).astype(np.float32)
    x[:, 7::13] = -np.inf
    x[:, 9::17] = np.nan
    at = np.where(np.arange(rows) % 2 == 0, 0, vocab - 1)
    x[np.arange(rows), at] = top
    t = np.full(rows, step * np.spacing(np.abs(top)))
    near = np.where(at == 0, np.float32(1 - 2.0 ** -24), np.float32(1e-6))
    for settings in ({}, {"top_k": np.full(rows, 3)}, {"top_p": np.full(rows, 0.9)}, {"min_p": np.full(rows, 1e-6)}):
        for u in (near, 1 - near, np.full(rows, 0.5)):
            assert draw(x, u, temperature=t, **settings).tolist() == at.tolist(), settings


@pytest.mark.parametrize("rows", [1, 8, 70, 200])
@pytest.mark.parametrize("exponent", [-119, -125, -135, -142])
def test_tiny_logits_and_temperatures(rows, exponent):
    """Logits and temperature scaled by a power of two, down to subnormal ones, draw what the
    unscaled ones do: only their quotient counts.  (Logits are multiples of 2^-6: exact.)"""
    vocab = 70001
    rng = np.random.default_rng(rows - exponent)
    x = np.round(rng.standard_normal((rows, vocab)) * 200).astype(np.float32) / 64
    scaled = np.ldexp(x, exponent)
    assert np.array_equal(np.ldexp(scaled.astype(np.float64), -exponent), x)
    temperature = rng.choice([0.25, 0.5, 1.0, 2.0], rows).astype(np.float32)
    for s in ({}, {"top_k": rng.integers(1, 3000, rows)}, {"top_p": rng.choice([0.3, 0.9], rows)},
              {"min_p": rng.choice([0.05, 0.3, 0.999], rows)}):
        u, want = rng.random(rows).astype(np.float32), np.zeros(rows, int)
        for r in range(rows):
            one = {k: (int if k == "top_k" else np.float32)(v[r]) for k, v in s.items()}
            want[r], near = sample_row(x[r], u[r], temperature[r], **one)
            while near <= vocab * 2.0 ** -43:  # the weights' rounding decides: another draw
                u[r] = rng.random()
                want[r], near = sample_row(x[r], u[r], temperature[r], **one)
        got = draw(scaled, u, temperature=np.ldexp(temperature, exponent), **s)
        assert got.tolist() == want.tolist(), s.keys()


@pytest.mark.parametrize("rows", [1, 8, 70, 200])
@pytest.mark.parametrize("temperature", [3e37, 1e38, np.inf])
def test_logits_further_apart_than_the_type_reaches(rows, temperature):
    """The row's range and 33 temperatures both pass the largest FP32 number; the cut lies
    among the far logits."""
    vocab = 70001
    rng = np.random.default_rng(rows)
    x = (rng.choice([-1, 1, 1, 1], (rows, vocab)) * rng.uniform(2e38, 3.3e38, (rows, vocab))).astype(np.float32)
    t = np.full(rows, temperature)
    for s in ({}, {"top_k": np.full(rows, vocab - 500)}, {"top_p": np.full(rows, 0.999)},
              {"top_k": np.full(rows, 60000), "top_p": np.full(rows, 0.98)}):
        # equal weights: the borders are multiples of one of them, and u lies between
        u = ((rng.integers(0, 60000, rows) + 0.5) / 60000).astype(np.float32)
        got = draw(x, u, temperature=t, **s)
        for r in range(rows):
            one = {k: (int if k == "top_k" else np.float32)(v[r]) for k, v in s.items()}
            want, near = sample_row(x[r], u[r], np.float32(temperature), **one)
            if near > vocab * 2.0 ** -43:
                assert got[r] == want, (r, one, int(got[r]), want)
            else:
                assert 0 <= got[r] < vocab


@pytest.mark.parametrize("rows", [63, 64, 95, 96, 191, 192])
@pytest.mark.parametrize("vocab", [32768, 32769])
def test_rows_agree_on_both_sides_of_every_size(rows, vocab):
    """A row's token is the same in the form that its batch takes and in that of a few rows."""
    rng = np.random.default_rng(rows)
    x = np.round(rng.standard_normal((rows, vocab)) * 3, 1).astype(np.float32)  # with equal logits
    u = rng.random(rows)
    s = {"temperature": rng.choice([0.5, 1.0], rows), "top_k": rng.choice([0, 40, 900], rows),
         "top_p": rng.choice([0.5, 0.9, 1.0], rows), "min_p": rng.choice([0.0, 0.05], rows)}
    few = np.concatenate([draw(x[i:i + 30], u[i:i + 30], **{k: v[i:i + 30] for k, v in s.items()})
                          for i in range(0, rows, 30)])
    assert np.array_equal(draw(x, u, **s), few)


def test_rows_behind_four_gigabytes():
    """Rows that start past 2^32 bytes and 2^31 logits of a tensor give what they give alone."""
    rows, vocab = 17000, 128256
    assert rows * vocab > 1 << 31
    x = torch.zeros((rows, vocab), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    some = [0, 8371, 8372, 16743, 16744, 16999]
    for r in some:
        x[r] = torch.randn(vocab, generator=gen, device="cuda") * 2.5
    u = torch.rand(rows, generator=gen, device="cuda")
    k = torch.full((rows,), 40, dtype=torch.int32, device="cuda")
    got = ops.sample_tokens(x, u, top_k=k)
    alone = [int(ops.sample_tokens(x[r:r + 1].clone(), u[r:r + 1].clone(), top_k=k[:1])) for r in some]
    assert got[some].tolist() == alone
