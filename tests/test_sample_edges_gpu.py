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
