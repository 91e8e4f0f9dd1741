"""The operators around the pick at the ends of their domains, on the GPU."""
import numpy as np
import pytest

import verbo_amd as V
from helpers import log, mode_ctx
from test_logits_ops import dev

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module")
def ctx():
    import torch

    assert torch.cuda.is_available(), "the gpu tests need a ROCm device"
    return mode_ctx()


# ---- infinities and NaN among the logits ---------------------------------------------------------------


def plain_ranks(x, ids):
    """How many ids come before each asked one; comparisons with NaN are false."""
    with np.errstate(invalid="ignore"):
        return np.array([[-1 if not 0 <= i < x.shape[1] else (x[r] > x[r, i]).sum() + (x[r, :i] == x[r, i]).sum() for i in row]
                         for r, row in enumerate(ids)])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,n", [(3, 700), (3, 4096), (3, 20001), (1100, 3001)])
def test_ranks_next_to_infinity(ctx, B, n, dtype):
    """One, two and many +inf before, among and after the asked ids, which lie above and below the few largest finite
    logits of a step; rows in one part and in several."""
    rng = np.random.default_rng(n)
    x = rng.normal(0, 3, (B, n)).astype(np.float32)
    x[0, 5] = INF
    x[1, [n // 3, n - 1]] = INF
    x[2, rng.integers(0, n, n // 20)] = INF
    for r in range(3, B):
        x[r, rng.integers(0, n, r % 4)] = INF
    xd = dev(x, dtype)
    xs = xd.float().cpu().numpy()
    top = np.argsort(-xs, 1, kind="stable")[:, 2:12]
    ids = np.concatenate([top, np.tile([0, 5, 200, 250, n // 3, n // 3 + 1, n - 2, n - 1, -1, n], (B, 1)), rng.integers(0, n, (B, 40))],
                         1).astype(np.int32)
    log("ranks", B, n, dtype)
    _, rank, _ = ctx.logprobs(xd, dev(ids))
    assert np.array_equal(rank.cpu().numpy(), plain_ranks(xs, ids))
