"""Token sampling on the GPU against the definition in 64 bits.  Weights are
held to 2^-44 of the largest, so a draw whose border is further off than
vocab * 2^-44 has one answer; the tests' draws are checked to be such."""
import numpy as np
import pytest
import torch

from sample_oracle import sample_row
from vllm_b200 import ops

pytestmark = pytest.mark.gpu


def run(x, u, **settings):
    dev = {k: None if v is None else torch.tensor(np.asarray(v, np.int32 if k == "top_k" else np.float32)).cuda()
           for k, v in settings.items()}
    xs = x if isinstance(x, torch.Tensor) else torch.from_numpy(np.asarray(x, np.float32)).cuda()
    got = ops.sample_tokens(xs, torch.tensor(np.asarray(u, np.float32)).cuda(), **dev)
    return got.cpu().numpy()


def check(x, u, got=None, **settings):
    got = run(x, u, **settings) if got is None else got
    for r in range(len(x)):
        one = {k: (np.float32 if k != "top_k" else int)(v[r]) for k, v in settings.items() if v is not None}
        want, near = sample_row(x[r], np.float32(u[r]), **one)
        assert near > x.shape[1] * 2.0 ** -43 or near == 0, (r, near)
        assert got[r] == want, (r, one, float(u[r]), int(got[r]), want)
    return got


def settings_of(rng, rows, k_hi):
    return {"temperature": rng.choice([0.1, 0.6, 1.0, 2.5], rows), "top_k": rng.integers(0, k_hi + 1, rows),
            "top_p": rng.choice([0.05, 0.5, 0.9, 0.999, 1.0], rows), "min_p": rng.choice([0.0, 0.0, 0.01, 0.3], rows)}


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 32, 33, 127, 1000, 4097, 32000, 50257, 128256, 150001])
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_random_rows(vocab, rows):
    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    for _ in range(3):
        check(x, rng.random(rows), **settings_of(rng, rows, min(vocab, 500)))


@pytest.mark.parametrize("vocab", [65535, 65536, 65539, 327680])
@pytest.mark.parametrize("rows", [1, 4])
def test_few_rows_of_large_vocabularies(vocab, rows):
    """Both sides of the sizes where a row gets the larger cluster."""
    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    x[:, rng.integers(0, vocab, 20)] += 8
    x[0, 1::2] = np.round(x[0, 1::2])  # ties at every cut
    for k_hi in (200, 5000):
        check(x, rng.random(rows), **settings_of(rng, rows, k_hi))
    check(x, rng.random(rows), top_p=np.full(rows, 0.9))
    check(x, rng.random(rows), top_k=np.full(rows, 3000), min_p=np.full(rows, 0.01))


@pytest.mark.parametrize("k", [160, 161, 223, 224, 225, 256, 257])
def test_top_k_around_the_lists_sizes(k):
    rng = np.random.default_rng(k)
    for rows in (2, 80, 200):
        x = (rng.standard_normal((rows, 30000)) * 2).astype(np.float32)
        x[::2] = np.round(x[::2] * 8) / 8  # ties
        check(x, rng.random(rows), top_k=np.full(rows, k), top_p=rng.choice([1.0, 0.8], rows))


def test_many_rows():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((300, 2000)) * 2).astype(np.float32)
    check(x, rng.random(300), **settings_of(rng, 300, 100))


def test_more_rows_than_are_put_in_turn_at_once():
    rng = np.random.default_rng(13)
    x = (rng.standard_normal((1100, 900)) * 2).astype(np.float32)
    check(x, rng.random(1100), **settings_of(rng, 1100, 400))


@pytest.mark.parametrize("only", ["temperature", "top_k", "top_p", "min_p", None])
def test_each_setting_alone_of_many_rows(only):
    rng = np.random.default_rng(14)
    x = (rng.standard_normal((200, 3000)) * 2).astype(np.float32)
    s = settings_of(rng, 200, 400)
    check(x, rng.random(200), **({only: s[only]} if only else {}))


@pytest.mark.parametrize("only", ["temperature", "top_k", "top_p", "min_p", None])
def test_each_setting_alone(only):
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((16, 5000)) * 2).astype(np.float32)
    s = settings_of(rng, 16, 60)
    check(x, rng.random(16), **({only: s[only]} if only else {}))


def test_ties_go_to_the_lowest_index():
    """Few distinct values: the cut of top-k and top-p lies among equal logits."""
    rng = np.random.default_rng(5)
    x = rng.integers(-3, 4, (64, 3001)).astype(np.float32)
    x[:, ::7] *= 0.0  # +0 and -0 are one value
    check(x, rng.random(64), top_k=rng.integers(1, 1500, 64))
    # equal weights: borders are multiples of one weight, uniforms lie between them
    flat = np.zeros((40, 1000), np.float32)
    check(flat, (rng.integers(0, 1000, 40) + 0.5) / 1000)
    check(flat, (rng.integers(0, 37, 40) + 0.5) / 37, top_k=np.full(40, 37))
    got = run(flat, np.full(40, 0.999999), top_p=np.full(40, 0.2505, np.float32))
    assert (got == 250).all()


def test_a_token_is_hit_in_proportion_to_its_weight():
    """An even sweep of uniforms over a small row hits each kept token as often as its share."""
    x = np.log(np.array([[4, 1, 2, 0.5, 8, 0.25]], np.float32)).repeat(4096, 0)
    u = (np.arange(4096) + 0.5) / 4096
    got = run(x, u, top_k=np.full(4096, 4))
    share = np.bincount(got, minlength=6) / 4096
    assert np.abs(share - np.array([4, 1, 2, 0, 8, 0]) / 15).max() <= 2 / 4096


@pytest.mark.parametrize("copies", [1, 9])
def test_masked_logits(copies):
    """-inf, NaN, the type's lowest value and rows without anything, in a few rows and in many."""
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((8, 700)) * 2).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 1:] = -np.inf
    x[3, ::2] = np.nan
    x[4, :350] = -np.inf
    x[5] = np.finfo(np.float32).min
    x[6, 5] = np.inf
    x[6, 600] = np.inf
    x[7, :699] = np.finfo(np.float32).min
    s = {"temperature": np.full(8, 0.8), "top_k": np.full(8, 650), "top_p": np.full(8, 0.95)}
    for u in (0.0, 0.3, 0.77):
        many = run(np.tile(x, (copies, 1)), np.full(8 * copies, u), **{k: np.tile(v, copies) for k, v in s.items()})
        assert np.array_equal(many, np.tile(many[:8], copies))
        got = check(x, np.full(8, u), got=many[:8], **s)
        assert got[0] == got[1] == -1 and got[2] == 0 and got[7] == 699
        assert got[3] % 2 == 1 and got[4] >= 350 and got[6] in (5, 600)
    greedy = run(x, np.full(8, 0.5), temperature=np.zeros(8))
    assert greedy.tolist()[:3] == [-1, -1, 0] and greedy[6] == 5 and greedy[5] == 0


def test_zero_temperature_is_the_largest_logit():
    rng = np.random.default_rng(7)
    x = rng.integers(0, 50, (9, 4000)).astype(np.float32)
    got = run(x, rng.random(9), temperature=np.zeros(9), top_k=np.full(9, 3), top_p=np.full(9, 0.1))
    assert np.array_equal(got, x.argmax(1))


def test_settings_at_and_past_their_ends():
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((1, 900)) * 2).astype(np.float32)
    best = int(x.argmax())
    assert run(x, [0.9], top_p=[0.0])[0] == best
    assert run(x, [0.9], top_p=[-1.0])[0] == best
    assert run(x, [0.9], min_p=[1.0])[0] == best
    assert run(x, [0.9], min_p=[7.0])[0] == best
    assert run(x, [0.9], top_k=[1])[0] == best
    assert run(x, [0.9], temperature=[1e-30])[0] == best
    assert run(x, [0.9], temperature=[np.nan])[0] == best
    free = run(x, [0.4])[0]
    for off in ({"top_k": [-5]}, {"top_k": [900]}, {"top_k": [2 ** 31 - 1]}, {"top_p": [1.0]}, {"top_p": [np.nan]},
                {"top_p": [2.0]}, {"min_p": [np.nan]}, {"min_p": [-1.0]}, {"temperature": [1.0]}):
        assert run(x, [0.4], **off)[0] == free, off
    assert run(x, [-3.0])[0] == run(x, [0.0])[0] == run(x, [np.nan])[0] == 0
    assert run(x, [1.0])[0] == run(x, [5.0])[0] == 899
    # an infinite temperature is an even draw
    assert run(x, [0.5005], temperature=[np.inf])[0] == 450


@pytest.mark.parametrize("rows", [7, 80])
def test_strided_and_unaligned_rows(rows):
    rng = np.random.default_rng(9)
    big = torch.from_numpy((rng.standard_normal((rows, 3010)) * 2).astype(np.float32)).cuda()
    for start, width in ((0, 3010), (1, 3000), (3, 2999), (2, 17)):
        x = big[:, start:start + width]
        u = rng.random(rows)
        s = settings_of(rng, rows, width // 2)
        check(x.cpu().numpy(), u, got=run(x, u, **s), **s)


def test_one_row_and_many_rows_agree():
    """A row's token does not depend on how many rows are drawn with it (two forms of the kernel)."""
    rng = np.random.default_rng(11)
    x = np.round(rng.standard_normal((90, 20011)) * 3, 1).astype(np.float32)  # with equal logits
    u, s = rng.random(90), settings_of(rng, 90, 9000)
    many = run(x, u, **s)
    few = np.concatenate([run(x[i:i + 9], u[i:i + 9], **{k: v[i:i + 9] for k, v in s.items()})
                          for i in range(0, 90, 9)])
    assert np.array_equal(many, few)


def test_repeats_bit_for_bit_and_captures():
    rng = np.random.default_rng(10)
    x = torch.from_numpy((rng.standard_normal((20, 30000)) * 2).astype(np.float32)).cuda()
    u = torch.rand(20, device="cuda")
    p = torch.full((20,), 0.9, device="cuda")
    want = ops.sample_tokens(x, u, top_p=p)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_tokens(x, u, top_p=p, out=out)
    for _ in range(5):
        out.fill_(-9)
        graph.replay()
        assert torch.equal(out, want)
    x2 = x.flip(1).contiguous()
    want2 = ops.sample_tokens(x2, u, top_p=p)
    x.copy_(x2)
    graph.replay()
    assert torch.equal(out, want2)
