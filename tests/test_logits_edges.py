"""The operators around the pick at the ends of their domains, on the GPU."""
import numpy as np
import pytest

import verbo_amd as V
from helpers import log, mode_ctx
from test_logits_ops import dev, plain_logprobs

pytestmark = pytest.mark.gpu

INF = float("inf")
NAN = float("nan")


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


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7, 4096, 4099, 60001])
def test_logprobs_of_rows_with_nan_or_infinity(ctx, n, dtype):
    """A row with a NaN or a +inf has no probabilities: its lse and its ids' log-probabilities are NaN, wherever the
    NaN lies and whatever surrounds it (a mask's -inf, nothing but NaN); ids outside the vocabulary are -inf as
    ever, the other rows of the batch are what they are without it, and NaN comes before no id."""
    rng = np.random.default_rng(n)
    at = sorted({0, n // 3, n - 1})
    rows, bad = [], []
    for fill in ("finite", "masked", "all"):
        for i in at:
            r = rng.normal(0, 3, n).astype(np.float32) if fill == "finite" else np.full(n, -INF if fill == "masked" else NAN, np.float32)
            r[i] = NAN
            rows.append(r)
            bad.append(True)
            rows.append(rng.normal(0, 3, n).astype(np.float32))
            bad.append(False)
    for i in at:
        r = rng.normal(0, 3, n).astype(np.float32)
        r[i] = INF
        rows.append(r)
        bad.append(True)
    r = np.full(n, -INF, np.float32)  # what a mask may leave: one allowed token and one NaN
    r[0], r[n - 1] = 1.0, NAN
    rows += [r, np.full(n, -INF, np.float32)]
    bad = np.array(bad + [True, False])
    xd = dev(np.array(rows), dtype)
    xs = xd.float().cpu().numpy()
    ids = np.tile(np.array(at + [n // 2, -1, n], np.int32), (len(rows), 1))
    inside = (ids >= 0) & (ids < n)
    log("nan", n, dtype)
    lp, rank, lse = (t.cpu().numpy() for t in ctx.logprobs(xd, dev(ids)))
    assert np.isnan(lse[bad]).all() and not np.isnan(lse[~bad]).any()
    assert np.isnan(lp[bad[:, None] & inside]).all()
    assert (lp[~inside] == -INF).all() and not np.isnan(lp[~bad]).any()
    assert np.array_equal(rank, plain_ranks(xs, ids))
    xs[bad] = 0.0  # the other rows beside ordinary ones
    again = ctx.logprobs(dev(xs, dtype), dev(ids))
    for a, b in zip((lp, rank, lse), again):
        assert np.array_equal(a[~bad], b.cpu().numpy()[~bad])
    wl, _, wz, tol = plain_logprobs(xs[~bad], ids[~bad])
    fin = np.isfinite(wz)
    z = lse[~bad]
    assert np.array_equal(z[~fin], wz[~fin]) and (np.abs(z[fin] - wz[fin]) <= (tol[fin] + 2.0 ** -24 * np.abs(wz[fin]))).all()
