"""The operators around the pick on the GPU (include/vsmp_logits.h): adjusted logits, log-probabilities and ranks, the
LM head with 4-bit weights, each against a plain implementation in 64 bits at the sizes, strides and masks where it
can go wrong; then all of them in a row, eagerly, from a replayed graph and on other streams.

Tolerances count roundings: u = 2^-24 is the most that rounding to fp32 takes, relative to the value."""
import numpy as np
import pytest

import verbo_amd as V
from helpers import Run, csr, log, mode_ctx
from verbo_amd import decode

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")
HALF = {"f32": None, "bf16": "bfloat16", "f16": "float16"}


@pytest.fixture(scope="module")
def ctx():
    import torch

    assert torch.cuda.is_available(), "the gpu tests need a ROCm device"
    return mode_ctx()


def dev(a, dtype=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(getattr(torch, HALF[dtype])) if dtype and HALF[dtype] else t


def strided(t, ld, shift=0):
    """The matrix t as a view with rows ld elements apart that starts `shift` elements into its memory."""
    import torch

    B, n = t.shape
    buf = torch.full((shift + B * ld,), 7.0 if t.is_floating_point() else 7, dtype=t.dtype, device=t.device)
    v = buf[shift:shift + B * ld].view(B, ld)[:, :n]
    v.copy_(t)
    return v


# ---- adjusted logits -----------------------------------------------------------------------------------


def plain_adjust(x, pens, hists=None, prompts=None, biases=None, masks=None):
    """(y, bound): the adjusted rows in 64 bits, and what three roundings to fp32 and the penalty's two may move."""
    y = x.astype(np.float64).copy()
    tol = np.zeros(y.shape)
    n = y.shape[1]
    for r in range(y.shape[0]):
        p = pens[r if len(pens) > 1 else 0]
        at = y[r].copy()
        with np.errstate(invalid="ignore", over="ignore"):
            if hists is not None:
                h = np.asarray(hists[r], np.int64)
                first = max(0, len(h) - p.window) if p.window > 0 else 0
                pos = np.arange(len(h))
                ok = (h >= 0) & (h < n) & (pos >= first)
                seen = np.unique(h[ok])
                at[seen] = np.where(at[seen] > 0, at[seen] / float(np.float32(p.repeat)), at[seen] * float(np.float32(p.repeat)))
                tol[r, seen] += U * np.abs(at[seen])
                made, c = np.unique(h[ok & (pos >= (prompts[r] if prompts is not None else 0))], return_counts=True)
                d = float(np.float32(p.presence)) + float(np.float32(p.frequency)) * c
                tol[r, made] += U * (2 * np.abs(float(np.float32(p.frequency)) * c) + np.abs(d) + np.abs(at[made] - d))
                at[made] -= d
            if biases is not None:
                for i, b in dict(biases[r]).items():
                    if 0 <= i < n:
                        at[i] += float(np.float32(b))
                        tol[r, i] += U * np.abs(at[i])
        at = np.where(np.isneginf(y[r]), y[r], at)
        if masks is not None and masks[r] is not None:
            at = np.where(masks[r], at, -INF)
        y[r] = at
    return y, 1.001 * tol


def pack(masks, n, words):
    out = np.zeros((len(masks), words), np.uint32)
    for m, a in enumerate(masks):
        bits = np.zeros(words * 32, bool)
        bits[:n] = a
        out[m] = np.packbits(bits, bitorder="little").view(np.uint32)
    return out.view(np.int32)


def check_adjusted(got, left, want, tol):
    g = got.cpu().numpy().astype(np.float64)
    assert g.shape == want.shape
    same = (g == want) | (np.isnan(g) & np.isnan(want))
    fin = np.isfinite(want)
    assert np.isfinite(g[fin]).all()
    assert same[~fin].all(), "an infinity or NaN is not where it should be"
    err = np.abs(np.where(fin, g, 0) - np.where(fin, want, 0))
    assert (err <= tol)[fin].all(), float(np.max(err[fin] - tol[fin]))
    with np.errstate(invalid="ignore"):
        assert np.array_equal(left.cpu().numpy(), (want > -INF).sum(1))


def bias_csr(biases):
    flat, off = csr([[i for i, _ in b] for b in biases])
    return dev(flat), dev(np.array([v for b in biases for _, v in b], np.float32)), dev(off)


def adjust_case(seed, B, n, hist=0, biases=0):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 3, (B, n)).astype(np.float32)
    x[rng.random((B, n)) < 0.02] = -INF
    x[rng.random((B, n)) < 0.02] = 0.0
    x[rng.random((B, n)) < 0.02] = -0.0
    hot = rng.integers(0, n, 5)
    hists = [np.where(rng.random(k) < 0.5, rng.choice(hot, k), rng.integers(-2, n + 2, k)).astype(np.int32)
             for k in rng.integers(0, hist + 1, B)]
    bias = [[(int(i), float(v)) for i, v in zip(np.where(rng.random(k) < 0.3, rng.choice(hot, k), rng.integers(-2, n + 2, k)),
                                                rng.choice([-100.0, 2.5, -0.75, 100.0, -INF], k))]
            for k in rng.integers(0, biases + 1, B)]
    return rng, x, hists, bias


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 2, 3, 31, 33, 4095, 4096, 4097, 8195, 20000])
def test_adjust_everything(ctx, n, dtype):
    """Penalties of each row's own with windows and prompts, biases that name an id twice, masks (none, some,
    nothing, beyond the table) on rows of any alignment."""
    import torch

    log("adjust", n, dtype)
    B = 6
    rng, x, hists, bias = adjust_case(n, B, n, 300, 40)
    hists[1] = np.zeros(0, np.int32)
    hists[2] = np.full(700, n - 1, np.int32)  # one id again and again
    bias[3] = [(0, 1.0), (n - 1, 2.0), (0, -3.0)]
    xd = dev(x, dtype)
    pens = [V.Penalty(1.3, 0.5, 0.25, w) for w in (0, 10, 64, 1, -5)] + [V.Penalty(0.8, -0.5, 0.0, 100)]
    prompts = np.array([len(h) // 2 for h in hists], np.int32)
    table = [rng.random(n) < 0.5, np.zeros(n, bool), np.ones(n, bool)]
    row = np.array([-1, 0, 0, 1, 2, 3], np.int32)
    masks = [None if m < 0 else table[m] if m < 3 else np.zeros(n, bool) for m in row]
    words = (n + 31) // 32 + 2
    ids, vals, boff = bias_csr(bias)
    h, off = csr(hists)
    left = torch.empty(B, dtype=torch.int32, device="cuda")
    want, tol = plain_adjust(xd.float().cpu().numpy(), pens, hists, prompts, bias, masks)
    for ld, shift in ((n, 0), (n + 1, 1), (n + 3, 3)):
        out = strided(torch.zeros(B, n, device="cuda"), n + 5, ld - n)
        around = out._base.clone()
        got = ctx.adjust_logits(strided(xd, ld, shift), V.to_device_penalties(pens), dev(h if h.size else np.zeros(1, np.int32)),
                                dev(off), dev(prompts), ids, vals, boff, dev(pack(table, n, words)), dev(row), out=out, left=left)
        assert got is out
        check_adjusted(got, left, want, tol)
        after = out._base.clone()  # nothing but the rows' own columns is written
        out.zero_()
        assert torch.equal(out._base, around), (ld, shift)
        assert not torch.equal(after, around) or n == 1


def test_adjust_rounds_each_step(ctx):
    """The adjustments are rounded one by one, the product before it is added: the bits of numpy's fp32."""
    n = 3000
    rng = np.random.default_rng(14)
    x = rng.normal(0, 3, (1, n)).astype(np.float32)
    h = rng.integers(0, n, 9000).astype(np.int32)
    b = rng.normal(0, 1, n).astype(np.float32)
    pen = V.Penalty(1.3, 0.37, 0.11, 0)
    got = ctx.adjust_logits(dev(x), pen, dev(h), dev(np.array([0, 9000], np.int32)), bias_ids=dev(np.arange(n, dtype=np.int32)), bias=dev(b),
                            bias_off=dev(np.array([0, n], np.int32)))
    f = np.float32
    c = np.bincount(h, minlength=n).astype(f)
    y = np.where(c > 0, np.where(x[0] > 0, x[0] / f(1.3), x[0] * f(1.3)), x[0])
    y = np.where(c > 0, y - (f(0.37) + f(0.11) * c), y) + b
    assert y.dtype == f and np.array_equal(got[0].cpu().numpy(), y)


@pytest.mark.parametrize("what", ["copy", "repeat", "presence", "frequency", "bias", "mask", "hist_off_penalty"])
def test_adjust_one_thing_at_a_time(ctx, what):
    """Each adjustment alone with shared penalties, and none at all (a copy); the others' arguments absent."""
    import torch

    B, n = 3, 5001
    rng, x, hists, bias = adjust_case(9, B, n, 200, 20)
    pen = {"repeat": V.Penalty(1.7), "presence": V.Penalty(presence=0.5), "frequency": V.Penalty(frequency=0.3, window=50),
           "hist_off_penalty": V.Penalty()}.get(what)
    h, off = csr(hists)
    masks = [rng.random(n) < 0.3 for _ in range(B)]
    left = torch.empty(B, dtype=torch.int32, device="cuda")
    kw = {}
    if pen is not None:
        kw.update(hist=dev(h), hist_off=dev(off))
    if what == "bias":
        kw.update(zip(("bias_ids", "bias", "bias_off"), bias_csr(bias)))
    if what == "mask":
        kw.update(mask=dev(pack(masks, n, (n + 31) // 32)))
    log("adjust", what)
    got = ctx.adjust_logits(dev(x), pen, left=left, **kw)
    want, tol = plain_adjust(x, [pen or V.Penalty()], hists if pen else None, None, bias if what == "bias" else None,
                             masks if what == "mask" else None)
    check_adjusted(got, left, want, tol)
    assert got.stride(0) % 4 == 0
    without = ctx.adjust_logits(dev(x), pen, **kw)  # and without the count
    assert np.array_equal(without.cpu().numpy(), got.cpu().numpy())


def test_adjust_forbidden_logits_may_be_anything(ctx):
    """NaN and infinities under the mask are -inf in the output; where they are allowed they stay; -inf stays -inf
    under a bias of +inf; a mask in the type's lowest value is an ordinary logit."""
    import torch

    n = 70
    x = np.zeros((2, n), np.float32)
    x[:, 0:4] = [np.nan, INF, -INF, np.finfo(np.float32).min]
    x[:, 40:44] = [np.nan, INF, -INF, np.finfo(np.float32).min]
    allow = np.ones((2, n), bool)
    allow[:, :4] = False
    left = torch.empty(2, dtype=torch.int32, device="cuda")
    got = ctx.adjust_logits(dev(x), mask=dev(pack(allow, n, 3)), left=left, bias_ids=dev(np.array([42, 2, 50], np.int32)),
                            bias=dev(np.array([INF, INF, INF], np.float32)), bias_off=dev(np.array([0, 3, 3], np.int32)))
    g = got.cpu().numpy()
    assert (g[:, :4] == -INF).all()
    assert np.isnan(g[:, 40]).all() and (g[:, 41] == INF).all() and (g[:, 42] == -INF).all()
    assert (g[:, 43] == np.finfo(np.float32).min).all()
    assert g[0, 50] == INF and g[1, 50] == 0.0
    assert left.cpu().tolist() == [n - 4 - 2] * 2  # not the NaN, not the -inf


def test_adjust_in_place_and_on_a_slice(ctx):
    """out = logits gives the same bits as another output; rows of a wider tensor keep what is behind them."""
    import torch

    B, n = 4, 9001
    _, x, hists, bias = adjust_case(3, B, n, 500, 50)
    h, off = csr(hists)
    wide = torch.full((B + 2, n + 7), 5.0, device="cuda")
    view = wide[1:1 + B, :n]
    view.copy_(dev(x))
    pen = V.Penalty(1.2, 0.1, 0.2, 0)
    kw = dict(hist=dev(h), hist_off=dev(off), **dict(zip(("bias_ids", "bias", "bias_off"), bias_csr(bias))))
    apart = ctx.adjust_logits(view, pen, **kw)
    got = ctx.adjust_logits(view, pen, out=view, **kw)
    assert got is view and np.array_equal(view.cpu().numpy(), apart.cpu().numpy())
    view.fill_(5.0)
    assert (wide == 5.0).all()


def test_adjust_many_rows(ctx):
    """More rows than one launch takes, with masks by row, histories and counts."""
    import torch

    B, n = 70000, 9
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (B, n)).astype(np.float32)
    masks = rng.random((B, n)) < 0.5
    h = rng.integers(0, n, B).astype(np.int32)
    words = np.zeros((B, 1), np.int32)
    for i in range(n):
        words[:, 0] |= masks[:, i].astype(np.int32) << i
    left = torch.empty(B, dtype=torch.int32, device="cuda")
    want = x.copy()
    np.add.at(want, (np.arange(B), h), -np.float32(0.5))
    want[~masks] = -INF
    off = np.arange(B + 1, dtype=np.int32)
    for kw in (dict(mask=dev(words)), dict(mask=dev(words[::-1]), mask_row=dev(np.arange(B - 1, -1, -1, dtype=np.int32)))):
        log("adjust", B, sorted(kw))
        got = ctx.adjust_logits(dev(x), V.Penalty(presence=0.5), dev(h), dev(off), left=left, **kw)
        assert np.array_equal(got.cpu().numpy(), want)
        assert np.array_equal(left.cpu().numpy(), masks.sum(1))
    pens = V.to_device_penalties(np.array([(1.0, 0.5, 0.0, 0)] * B, V.PENALTY_DTYPE))
    got = ctx.adjust_logits(dev(x), pens, dev(h), dev(off), mask=dev(words))
    assert np.array_equal(got.cpu().numpy(), want)


def test_adjust_long_histories(ctx):
    """Histories far longer than a part: counts above 2^16 of one id, and prompts that end inside."""
    import torch

    n = 12345
    rng = np.random.default_rng(4)
    x = rng.normal(0, 3, (2, n)).astype(np.float32)
    hists = [np.concatenate([np.full(70001, 77, np.int32), rng.integers(0, n, 30000).astype(np.int32)]),
             rng.integers(0, n, 50001).astype(np.int32)]
    h, off = csr(hists)
    prompts = np.array([1, 50000], np.int32)
    left = torch.empty(2, dtype=torch.int32, device="cuda")
    pen = V.Penalty(1.1, 0.5, 2.0 ** -10, 0)
    got = ctx.adjust_logits(dev(x), pen, dev(h), dev(off), dev(prompts), left=left)
    check_adjusted(got, left, *plain_adjust(x, [pen], hists, prompts))


def test_adjust_prompt_lengths_beyond_the_history(ctx):
    """A prompt length below 0 is none, one above the history's length is all of it, also at the type's ends."""
    n = 500
    x = np.zeros((4, n), np.float32)
    h = np.tile(np.arange(10, dtype=np.int32), 4)
    prompts = np.array([-(1 << 31), -1, (1 << 31) - 1, 11], np.int32)
    got = ctx.adjust_logits(dev(x), V.Penalty(presence=1.0), dev(h), dev(np.arange(0, 41, 10, dtype=np.int32)), dev(prompts)).cpu().numpy()
    want = np.zeros((4, n), np.float32)
    want[:2, :10] = -1.0
    assert np.array_equal(got, want)


def test_adjust_repeat_is_the_picks_penalty(ctx):
    """The multiplicative penalty applied here and the one inside the pick give the same picks, penalised logits
    included: 40 rows, greedy and sampled."""
    import torch

    B, n = 40, 30001
    rng = np.random.default_rng(6)
    x = strided(dev(rng.normal(0, 3, (B, n)).astype(np.float32)), 30004)
    hists = [rng.integers(0, n, int(k)).astype(np.int32) for k in rng.integers(0, 3000, B)]
    h, off = csr(hists)
    for fields in (dict(temp=0.0), dict(temp=0.8, top_k=50, top_p=0.95), dict(temp=1.0, top_k=0, top_p=0.9)):
        inside = V.Params(repeat=1.3, repeat_last=900, seed=5, **fields)
        after = V.Params(repeat=1.0, repeat_last=900, seed=5, **fields)
        info = [torch.zeros(B * 72, dtype=torch.uint8, device="cuda") for _ in range(2)]
        a = ctx.pick_batch(x, inside, dev(h), dev(off), info=info[0])
        y = ctx.adjust_logits(x, V.Penalty(repeat=1.3, window=900), dev(h), dev(off))
        b = ctx.pick_batch(y, after, info=info[1])
        assert np.array_equal(a.cpu().numpy(), b.cpu().numpy())
        assert np.array_equal(V.row_info(info[0])["mx"], V.row_info(info[1])["mx"])


# ---- log-probabilities -----------------------------------------------------------------------------------


def plain_logprobs(x, ids):
    """(logprob, rank, lse) of rows x in 64 bits, and the roundings' bound on the log of the sum: every exponential's
    argument is rounded three times (difference, product, the constant's own) and its value twice; the sums of one
    thread, of a wave, a workgroup and a row's parts follow one another (at most n / 256 + 64 additions and as many
    rescalings, one per step of 16 or more logits); the log is rounded once to two units."""
    x = x.astype(np.float64)
    B, n = x.shape
    lp, rank, lse, tol = np.full(ids.shape, -INF), np.full(ids.shape, -1), np.full(B, -INF), np.zeros(B)
    for r in range(B):
        m = x[r].max()
        if m > -INF:
            e = np.exp(x[r] - m)
            lse[r] = m + np.log(e.sum())
            p = e / e.sum()
            far = np.where(p > 0, np.abs(np.where(p > 0, x[r], m) - m), 0)
            tol[r] = U * (3 * (p * far).sum() + 4 + 2 * (n / 256 + 64) + 4 * np.abs(np.log(e.sum())))
        for j, i in enumerate(ids[r]):
            if 0 <= i < n:
                # not x_i - lse, which 64 bits cannot hold next to values of 1e38 (a row of one value has -log n)
                lp[r, j] = (x[r, i] - m) - np.log(e.sum()) if x[r, i] > -INF else -INF
                rank[r, j] = (x[r] > x[r, i]).sum() + (x[r, :i] == x[r, i]).sum()
    return lp, rank, lse, tol


def check_logprobs(ctx, x, ids, **kw):
    xs = x.float().cpu().numpy()
    lp, rank, lse = ctx.logprobs(x, dev(ids) if ids is not None else None, **kw)
    wl, wr, wz, tol = plain_logprobs(xs, ids if ids is not None else np.zeros((len(xs), 0), np.int32))
    z = lse.cpu().numpy()
    fin = np.isfinite(wz)
    assert np.array_equal(z[~fin], wz[~fin])
    assert (np.abs(z[fin] - wz[fin]) <= (tol + U * np.abs(wz))[fin]).all()
    if ids is None or ids.shape[1] == 0:
        return
    g = lp.cpu().numpy()
    fin = np.isfinite(wl)
    assert np.array_equal(g[~fin], wl[~fin])
    with np.errstate(invalid="ignore"):
        err, most = np.abs(g - wl), tol[:, None] + 2 * U * (np.abs(wl) + tol[:, None])
        most = most + U * np.abs(np.where(fin, np.take_along_axis(xs, np.clip(ids, 0, xs.shape[1] - 1), 1) - xs.max(1, keepdims=True), 0))
    assert (err <= most)[fin].all(), float(np.max((err - most)[fin]))
    if kw.get("rank", True):
        assert np.array_equal(rank.cpu().numpy(), wr)
    else:
        assert rank is None


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 2, 7, 63, 65, 4095, 4097, 8191, 8192, 8193, 50257])
def test_logprobs_match(ctx, n, dtype):
    """Ids at the ends of the row, the likeliest ones, the same one twice, outside the vocabulary; ties (every
    value of the 16-bit types occurs again and again); rows of any alignment; with and without ranks."""
    rng = np.random.default_rng(n)
    B = 5
    x = rng.normal(0, 4, (B, n)).astype(np.float32)
    x[1] = np.round(x[1])
    x[2] = 1.5
    x[3, rng.random(n) < 0.5] = -INF
    xd = dev(x, dtype)
    top = np.argsort(-xd.float().cpu().numpy(), 1, kind="stable")[:, :5]
    ids = np.concatenate([top, rng.integers(0, n, (B, 6)), np.tile([0, n - 1, n // 2, n // 2, -1, n, -(1 << 31), (1 << 31) - 1], (B, 1))],
                         1).astype(np.int32)
    log("logprobs", n, dtype)
    check_logprobs(ctx, xd, ids)
    check_logprobs(ctx, strided(xd, n + 1, 1), ids[:, :1])
    check_logprobs(ctx, strided(xd, n + 3, 3), ids, rank=False)
    check_logprobs(ctx, xd, None)
    check_logprobs(ctx, xd, ids[:, :0])


@pytest.mark.parametrize("B", [1, 3, 64, 300, 2500])
def test_logprobs_batches(ctx, B):
    """Batches that are cut into parts and ones that are not, 64 ids a row."""
    rng = np.random.default_rng(B)
    n = 20011 if B <= 300 else 3001
    x = rng.normal(0, 2, (B, n)).astype(np.float32)
    log("logprobs batch", B)
    check_logprobs(ctx, dev(x), rng.integers(0, n, (B, 64)).astype(np.int32))


def test_logprobs_extreme_rows(ctx):
    """A row of -inf alone, one with a single token left (probability 1), huge and tiny spreads, the type's lowest
    value as a mask, and logits whose exponentials under- or overflow unshifted."""
    n = 9000
    low = float(np.finfo(np.float32).min)
    x = np.full((7, n), -INF, np.float32)
    x[1, 4321] = -3.0
    x[2] = low
    x[2, 17] = 2.0
    x[3] = np.linspace(-1e30, 1e30, n)
    x[4] = 1e4
    x[5] = -1e4 + np.arange(n) % 3
    x[6] = low
    ids = np.tile(np.array([0, 17, 4321, n - 1], np.int32), (7, 1))
    check_logprobs(ctx, dev(x), ids)
    lp, rank, lse = ctx.logprobs(dev(x), dev(ids))
    assert (lp[0] == -INF).all() and lse[0] == -INF and rank[0].tolist() == [0, 17, 4321, n - 1]
    assert lp[1, 2] == 0.0 and lse[1] == -3.0
    assert lp[2, 1] == 0.0 and rank[2].tolist() == [1, 0, 4321, n - 1]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lanes", [1, 2, 4, 5, 16])
def test_logprobs_crowded_tops(ctx, dtype, lanes):
    """Large logits, with and without ties, that a few lanes of every lane row hold in all their groups: from a list
    that takes them to more than it holds and more lanes than it takes. Ids among them, between them and far below."""
    n, N = 20000, 4 if dtype == "f32" else 8
    rng = np.random.default_rng(lanes)
    x = rng.normal(0, 1, (4, n)).astype(np.float32)
    at = np.array([N * (16 * r + l + 256 * g) + k for r in range(4) for l in range(lanes) for g in range(4) for k in range(N)])
    x[0, at] = 10.0
    x[1, at] = 10.0 + rng.integers(0, 3, at.size)
    x[2, at] = np.linspace(8.0, 16.0, at.size)
    x[3, at] = 10.0 + rng.random(at.size)
    x[:, at + 1] = np.where(rng.random((4, at.size)) < 0.3, 9.0, x[:, at + 1])
    ids = np.concatenate([rng.choice(at, (4, 40)), rng.choice(at, (4, 10)) + 1, rng.integers(0, n, (4, 13)), np.full((4, 1), at[0])], 1)
    check_logprobs(ctx, dev(x, dtype), ids.astype(np.int32))


def test_logprobs_of_the_candidates(ctx):
    """The ids that pick_batch reports in order are at ranks 0, 1, 2, ... and the picked one at its info's rank."""
    import torch

    B, n, k = 20, 40000, 21
    rng = np.random.default_rng(8)
    x = dev(np.round(rng.normal(0, 3, (B, n)) * 8).astype(np.float32) / 8)  # with ties
    cand = torch.full((B, k), -1, dtype=torch.int32, device="cuda")
    pr = torch.zeros((B, k), dtype=torch.float64, device="cuda")
    info = torch.zeros(B * 72, dtype=torch.uint8, device="cuda")
    out = ctx.pick_batch(x, V.Params(temp=1.0, top_k=k, top_p=1.0, min_p=0.0, repeat=1.0, seed=3), info=info, cand_ids=cand, cand_pr=pr)
    lp, rank, _ = ctx.logprobs(x, torch.cat([out[:, None], cand], 1))
    assert np.array_equal(rank[:, 1:].cpu().numpy(), np.tile(np.arange(k), (B, 1)))
    assert np.array_equal(rank[:, 0].cpu().numpy(), V.row_info(info)["rank"])
    assert (lp[:, 1:].diff(dim=1) <= 0).all()


# ---- the head with 4-bit weights ---------------------------------------------------------------------------


def q4_weights(seed, n, D, G, scales="bf16", zeros=False):
    """(q, scales, zeros) on the device, and the weights in 64 bits."""
    rng = np.random.default_rng(seed)
    k = rng.integers(0, 16, (n, D))
    k[0] = 0
    k[-1] = 15
    q = (k[:, 0::2] | (k[:, 1::2] << 4)).astype(np.uint8)
    s = dev((rng.normal(0, 1, (n, D // G)) * 0.02).astype(np.float32), scales)
    z = rng.integers(0, 16, (n, D // G)).astype(np.uint8) if zeros else None
    if zeros:
        z[n // 2] = 255
    w = k - np.repeat(z.astype(np.int64) if zeros else np.full((n, D // G), 8), G, 1)
    return dev(q), s, dev(z) if zeros else None, w


def check_head(got, hidden, s, z, w, G):
    """Every logit within what the roundings may take: a group's matrix sums hold x (16 + q) and the offset
    -(16 + z) X on top of each other (G + 1 additions of at most two units each, X itself of log2 G + 1), and the
    groups' results are scaled and added, one rounding each."""
    import torch

    x = hidden.double().cpu()
    B, D = x.shape
    sd = s.double().cpu()
    off = 16.0 + (z.double().cpu() if z is not None else torch.full(sd.shape, 8.0, dtype=torch.float64))
    want = x @ (torch.from_numpy(w).double() * sd.repeat_interleave(G, 1)).t()
    ax = x.abs().reshape(B, D // G, G).sum(2)
    mass = ax @ (sd.abs() * (31.0 + off)).t()
    tol = U * (2 * (G + 1) + 10 + D // G + 1) * mass
    g = got.double().cpu()
    assert torch.isfinite(g).all()
    err = (g - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    # and far closer than that on the whole: a column or a group mixed up is off by the logits' own size
    assert float(err.norm()) <= 2e-6 * float(mass.norm())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("G,zeros,scales", [(32, False, "bf16"), (32, True, "f32"), (64, False, "f16"), (64, True, "bf16"),
                                            (128, False, "f32"), (128, True, "f16")])
def test_head_q4_sizes(ctx, G, zeros, scales, dtype):
    """Hidden sizes of one group up to several chunks, with blocks and chunks that end early; vocabularies around
    the tile's 128 columns; batches around its 16, 32 and 64 rows; padded strides."""
    rng = np.random.default_rng(G)
    for D in sorted({G, 3 * G, 5 * G, 640 // G * G, 512 + G, 1024, 1056 // G * G}):
        for n, B in ((1, 1), (15, 2), (17, 16), (128, 17), (129, 33), (300, 65), (127, 130)):
            q, s, z, w = q4_weights(D + n, n, D, G, scales, zeros)
            hidden = dev(rng.normal(0, 1, (B, D)).astype(np.float32) * rng.choice([0.1, 1, 8], (1, D)).astype(np.float32), dtype)
            log("head q4", G, D, n, B)
            got = ctx.head_logits_q4(hidden, q, s, G, zeros=z)
            check_head(got, hidden, s, z, w, G)
    out = strided(got.clone().zero_(), 131, 1)
    around = out._base.clone()
    again = ctx.head_logits_q4(strided(hidden, D + 8), strided(q, D // 2 + 16), strided(s, D // G + 3), G,
                               zeros=strided(z, D // G + 1) if zeros else None, logits=out)
    assert again is out and np.array_equal(out.cpu().numpy(), got.cpu().numpy())
    out.zero_()
    assert np.array_equal(out._base.cpu().numpy(), around.cpu().numpy())


@pytest.mark.parametrize("n,D,G,B,zeros", [(5000, 4096, 128, 3, True), (2049, 16384, 32, 3, True), (151936, 896, 64, 3, True),
                                           (333, 4096, 64, 40, False), (100, 16384, 32, 17, True), (257, 2240, 32, 64, True),
                                           (290, 2176, 128, 70, False), (65, 16256, 128, 16, True), (70, 8192, 64, 129, False)])
def test_head_q4_large(ctx, n, D, G, B, zeros):
    """Large vocabularies and hidden sizes; hidden states that do not fit on chip whole, in chunks that end early."""
    rng = np.random.default_rng(1)
    q, s, z, w = q4_weights(n, n, D, G, "bf16", zeros)
    hidden = dev(rng.normal(0, 1, (B, D)).astype(np.float32), "bf16")
    log("head q4", n, D, G, B)
    got = ctx.head_logits_q4(hidden, q, s, G, zeros=z)
    check_head(got, hidden, s, z, w, G)
    one = ctx.head_logits_q4(hidden[B - 1:], q, s, G, zeros=z)
    assert np.array_equal(one.cpu().numpy(), got[B - 1:].cpu().numpy())


@pytest.mark.parametrize("G,zeros", [(32, True), (64, False), (128, False)])
def test_head_q4_does_not_depend_on_the_batch(ctx, G, zeros):
    """A row's logits are the same bits alone and in batches of every tile shape, whatever shares them."""
    rng = np.random.default_rng(5)
    q, s, z, _ = q4_weights(3, 1000, 1408, G, "f16", zeros)
    hidden = dev(rng.normal(0, 1, (130, 1408)).astype(np.float32), "bf16")
    full = ctx.head_logits_q4(hidden, q, s, G, zeros=z).cpu().numpy()
    for a, b in ((0, 1), (129, 130), (5, 9), (7, 23), (40, 72), (64, 128), (50, 100)):
        assert np.array_equal(ctx.head_logits_q4(hidden[a:b], q, s, G, zeros=z).cpu().numpy(), full[a:b]), (a, b)


def test_head_q4_nibbles_and_scales(ctx):
    """Each weight alone: one-hot hidden states give back scale * (q - zero), exactly, in the weights' order."""
    import torch

    n, D, G = 40, 256, 64
    q, s, z, w = q4_weights(11, n, D, G, "f32", True)
    got = ctx.head_logits_q4(torch.eye(D, device="cuda").bfloat16(), q, s, G, zeros=z)
    assert torch.equal(got.t().contiguous().cpu(), torch.from_numpy(w).float() * s.cpu().repeat_interleave(G, 1))


# ---- far offsets -------------------------------------------------------------------------------------------


def test_offsets_beyond_32_bits(ctx):
    """Rows 2^30 elements apart: the last one starts beyond 2^31 elements of every operand that may lie so far out."""
    import torch

    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    ld, B, n = 1 << 30, 4, 300
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (B, n)).astype(np.float32)
    far = torch.empty(B * ld, dtype=torch.float16, device="cuda").view(B, ld)[:, :n]
    far.copy_(dev(x))
    out = torch.empty(B * ld, dtype=torch.float32, device="cuda").view(B, ld)[:, :n]
    near = far.contiguous()
    ids = dev(rng.integers(0, n, (B, 3)).astype(np.int32))
    got = ctx.adjust_logits(far, V.Penalty(presence=0.5), ids.reshape(-1).contiguous(), dev(np.arange(B + 1, dtype=np.int32) * 3), out=out)
    want = ctx.adjust_logits(near, V.Penalty(presence=0.5), ids.reshape(-1).contiguous(), dev(np.arange(B + 1, dtype=np.int32) * 3))
    assert torch.equal(got, want)
    for a, b in zip(ctx.logprobs(far, ids), ctx.logprobs(near, ids)):
        assert torch.equal(a, b)
    hidden, (q, s, z, w) = dev(rng.normal(0, 1, (B, 64)).astype(np.float32), "f16"), q4_weights(2, n, 64, 32)
    ctx.head_logits_q4(hidden, q, s, 32, logits=out)
    assert torch.equal(out, ctx.head_logits_q4(hidden, q, s, 32))


# ---- together --------------------------------------------------------------------------------------------


class Step:
    """One serving step: the 4-bit head, the adjustments, the pick and its log-probabilities, on buffers of its own."""

    def __init__(self, ctx, seed, B=6, n=5003, D=320):
        import torch

        self.ctx, self.B, self.n = ctx, B, n
        rng = np.random.default_rng(seed)
        self.q, self.s, self.z, self.w = q4_weights(seed, n, D, 64, "f16", True)
        self.hidden = dev(rng.normal(0, 1, (B, D)).astype(np.float32), "bf16")
        self.hists = [rng.integers(0, n, int(k)).astype(np.int32) for k in rng.integers(1, 400, B)]
        self.h, self.off = (dev(a) for a in csr(self.hists))
        self.masks = [None if r == 0 else rng.random(n) < 0.2 for r in range(B)]
        self.mask = dev(pack([m for m in self.masks if m is not None], n, (n + 31) // 32))
        self.mask_row = dev(np.arange(-1, B - 1, dtype=np.int32))
        self.pen = V.Penalty(1.2, 0.2, 0.1, 200)
        self.params = V.Params(temp=0.8, top_k=20, top_p=0.95, min_p=0.0, repeat=1.0, seed=seed)
        self.u = dev(rng.random(B))
        self.raw = torch.empty(B, (n + 3) // 4 * 4, device="cuda")[:, :n]
        self.x = torch.empty(B, (n + 3) // 4 * 4, device="cuda")[:, :n]
        self.left = torch.empty(B, dtype=torch.int32, device="cuda")
        self.ids = torch.empty(B, dtype=torch.int32, device="cuda")

    def run(self, stream=None):
        kw = dict(stream=stream)
        self.ctx.head_logits_q4(self.hidden, self.q, self.s, 64, zeros=self.z, logits=self.raw, **kw)
        self.ctx.adjust_logits(self.raw, self.pen, self.h, self.off, mask=self.mask, mask_row=self.mask_row, out=self.x, left=self.left, **kw)
        self.ctx.pick_batch(self.x, self.params, u_mode=V.U_SUPPLIED, u=self.u, out=self.ids, **kw)
        self.lp = self.ctx.logprobs(self.x, self.ids[:, None], **kw)
        return self

    def results(self):
        import torch

        torch.cuda.synchronize()
        return [t.cpu().numpy().copy() for t in (self.raw, self.x, self.left, self.ids, *self.lp)]


def same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert np.array_equal(x, y)


def test_a_serving_step(ctx):
    """The operators in a row: the head's logits and the adjustment against 64 bits, the picks against the oracle on
    the adjusted logits, the log-probabilities against 64 bits; no forbidden token is picked."""
    st = Step(ctx, 21).run()
    raw, x, left, ids, lp, rank, lse = st.results()
    check_head(st.raw, st.hidden, st.s, st.z, st.w, 64)
    want, tol = plain_adjust(raw, [st.pen], st.hists, None, None, st.masks)
    check_adjusted(st.x, st.left, want, tol)
    run = Run(ctx, x, V.params_array(n=1, temp=0.8, top_k=20, top_p=0.95, min_p=0.0, repeat=1.0, seed=21),
              u=st.u.cpu().numpy(), cand_cap=0)
    run.report()
    assert np.array_equal(run.ids, ids)
    for r, m in enumerate(st.masks):
        assert m is None or m[ids[r]]
    check_logprobs(ctx, st.x, ids[:, None])


def test_a_captured_serving_step(ctx):
    """The step captured after one eager call and replayed with new inputs, eager work of the same context between the
    replays: every replay gives the eager step's bits. A second graph of another context is replayed in turn."""
    import torch

    mine = V.Context(0)
    steps = [Step(mine, 31), Step(V.Context(0), 32, B=40, n=7001)]
    side = torch.cuda.Stream()
    graphs = []
    for st in steps:
        st.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            st.run(torch.cuda.current_stream())
        graphs.append(g)
    rng = np.random.default_rng(7)
    for rep in range(4):
        for k, (st, g) in enumerate(zip(steps, graphs)):
            st.hidden.copy_(dev(rng.normal(0, 1, st.hidden.shape).astype(np.float32), "bf16"))
            st.mask_row.copy_(st.mask_row.roll(1))
            held = st.lp
            g.replay()
            got = st.results()
            log("replay", rep, k)
            same(got, Step.results(st.run()))  # eagerly on the same inputs
            st.lp = held


def test_a_capture_needs_its_scratch_first():
    """A context that has no scratch yet refuses a captured call that needs it, with nothing launched, and takes
    the call once it was issued eagerly; calls that need none are captured at once."""
    import torch

    fresh = V.Context(0)
    x = torch.randn(2, 20000, device="cuda")
    ids = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    left = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    ones, boff = torch.ones(2, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    errors = []
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        for call in (lambda: fresh.logprobs(x, ids), lambda: fresh.adjust_logits(x, left=left, out=out)):
            try:
                call()
            except V.VsmpError as e:
                errors.append(str(e))
        fresh.adjust_logits(x, bias_ids=ids.reshape(-1), bias=ones, bias_off=boff, out=out)
    assert len(errors) == 2 and all("issue the call once" in e for e in errors)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:, 1:], x[:, 1:]) and torch.equal(out[:, 0], x[:, 0] + 1.0)
    fresh.logprobs(x, ids)
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2, stream=torch.cuda.Stream()):
        lp = fresh.logprobs(x, ids)
        fresh.adjust_logits(x, left=left, out=out)
    for _ in range(3):
        left.zero_()
        g2.replay()
        torch.cuda.synchronize()
        assert left.cpu().tolist() == [20000, 20000]
        assert torch.equal(lp[0], fresh.logprobs(x, ids)[0])


def test_streams_and_contexts(ctx):
    """Steps of two contexts on two streams at once, and of one context on a stream that waits for its last call."""
    import torch

    a, b = Step(V.Context(0), 41, B=30, n=9001), Step(V.Context(0), 42, B=3, n=40001)
    want = [st.run().results() for st in (a, b)]
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(sa):
            a.run()
        with torch.cuda.stream(sb):
            b.run()
    same(a.results(), want[0])
    same(b.results(), want[1])
    with torch.cuda.stream(sa):
        a.run()
    sb.wait_stream(sa)
    with torch.cuda.stream(sb):
        a.run()
    same(a.results(), want[0])


def test_same_inputs_same_bits(ctx):
    """Every operator gives the same bits again and again: no sum depends on the order in which parts arrive."""
    st = Step(ctx, 51, B=17, n=60001)
    first = st.run().results()
    for _ in range(5):
        same(st.run().results(), first)


# ---- the batched decoder -------------------------------------------------------------------------------------


def test_bsampler_adjusts_by_the_slots_histories(ctx):
    """Rows of a call are penalised by their slots' histories, in whatever order the slots are listed, as their
    histories grow; slots that are not listed stay as they are."""
    import torch

    n, slots = 3001, 7
    rng = np.random.default_rng(12)
    d = decode.BatchDecoder.with_slots(slots, n)
    stream = torch.cuda.current_stream()
    hists = {}
    for s in range(slots):
        ids = rng.integers(0, n, int(rng.integers(0, 50))).astype(np.int32)
        d.admit(s, V.Params(temp=0.0, repeat_last=0, repeat=1.0), ids, stream)
        hists[s] = ids.tolist()
    left = torch.empty(slots, dtype=torch.int32, device="cuda")
    for step, live in enumerate(([5, 0, 3], [1, 2], [6, 5, 4, 3, 2, 1, 0])):
        rows = dev(np.array(live, np.int32))
        x = rng.normal(0, 2, (len(live), n)).astype(np.float32)
        pens = [V.Penalty(1.0 + 0.1 * i, 0.5, 0.25, int(w)) for i, w in enumerate(rng.choice([0, 10], len(live)))]
        masks = [rng.random(n) < 0.5 for _ in live]
        y = d.adjust_rows(dev(x), rows, V.to_device_penalties(pens), mask=dev(pack(masks, n, (n + 31) // 32)), left=left)
        want, tol = plain_adjust(x, pens if len(pens) > 1 else pens, [hists[s] for s in live], None, None, masks)
        check_adjusted(y, left[:len(live)], want, tol)
        out = torch.empty(len(live), dtype=torch.int32, device="cuda")
        d.pick_rows(y, rows, out, stream)
        assert np.array_equal(out.cpu().numpy(), want.argmax(1))
        d.accept_rows(out, rows, torch.ones(len(live), dtype=torch.int32, device="cuda"), stream)
        for s, t in zip(live, out.cpu().tolist()):
            hists[s].append(t)
    with pytest.raises(V.VsmpError, match="rows"):
        d.adjust_rows(dev(x), dev(np.zeros(7, np.int64)))


def test_serve_with_penalties(ctx):
    """A serving loop whose requests carry penalties: greedy requests over constant logits. With a presence penalty
    above every gap a request never says a token twice; one without penalties always says the same."""
    import torch

    n = 500
    base = torch.linspace(5.0, 0.0, n, device="cuda")[None, :]
    reqs = [decode.Request([0], decode.Opts(max_tokens=6, temp=0.0), repeat_last=0, penalty=V.Penalty(presence=100.0)),
            decode.Request([0], decode.Opts(max_tokens=6, temp=0.0), repeat_last=0),
            decode.Request([3], decode.Opts(max_tokens=4, temp=0.0), repeat_last=0, arrival=2, penalty=V.Penalty(frequency=50.0))]
    res = decode.BatchDecoder.with_slots(2, n).serve(reqs, lambda js, steps, last: base.expand(len(js), n).contiguous())
    assert res[0][0] == [1, 2, 3, 4, 5, 6]
    assert res[1][0] == [0] * 6
    assert res[2][0] == [0, 1, 2, 4]
    plain = decode.BatchDecoder.with_slots(2, n).serve(
        [decode.Request([0], decode.Opts(max_tokens=6, temp=0.0), repeat_last=0)], lambda js, steps, last: base.expand(len(js), n).contiguous())
    assert plain[0][0] == [0] * 6


# ---- refusals on the device ----------------------------------------------------------------------------------


def test_refusals(ctx):
    import torch

    x = torch.zeros(2, 64, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    for call, words in [
        (lambda: ctx.adjust_logits(x.double()), "float32, bfloat16 or float16"),
        (lambda: ctx.adjust_logits(x[0]), "2-D"),
        (lambda: ctx.adjust_logits(x.t()), "contiguous rows"),
        (lambda: ctx.adjust_logits(x[:1].expand(2, 64)), "stride"),
        (lambda: ctx.adjust_logits(x, out=torch.empty(2, 63, device="cuda")), "shape"),
        (lambda: ctx.adjust_logits(x, out=x.bfloat16()), "float32"),
        (lambda: ctx.adjust_logits(x, hist=i), "go together"),
        (lambda: ctx.adjust_logits(x, hist=i, hist_off=i[:2]), "hist_off"),
        (lambda: ctx.adjust_logits(x, hist=i.long(), hist_off=i), "hist"),
        (lambda: ctx.adjust_logits(x, hist=i.cpu(), hist_off=i), "hist"),
        (lambda: ctx.adjust_logits(x, bias_ids=i, bias_off=i), "go together"),
        (lambda: ctx.adjust_logits(x, bias_ids=i, bias=i, bias_off=i), "bias"),
        (lambda: ctx.adjust_logits(x, bias_ids=i, bias=x[0, :2], bias_off=i), "bias"),
        (lambda: ctx.adjust_logits(x, mask=i[None, :1]), "mask"),
        (lambda: ctx.adjust_logits(x, mask=i[None, :2]), "mask of its own"),
        (lambda: ctx.adjust_logits(x, mask=i[None, :2], mask_row=i[:1]), "mask_row"),
        (lambda: ctx.adjust_logits(x, mask=i[:2].reshape(2, 1).expand(2, 2)), "mask"),
        (lambda: ctx.adjust_logits(x, left=i[:1]), "left"),
        (lambda: ctx.adjust_logits(x, V.Penalty(repeat=0.0)), "repeat above 0"),
        (lambda: ctx.adjust_logits(x, torch.zeros(16, dtype=torch.uint8, device="cuda")), "B entries"),
        (lambda: ctx.logprobs(x, torch.zeros(2, 65, dtype=torch.int32, device="cuda")), "0 <= n <= 64"),
        (lambda: ctx.logprobs(x, i[None, :1]), "ids"),
        (lambda: ctx.logprobs(x, i[:2, None].long()), "ids"),
        (lambda: ctx.head_logits_q4(x, i, i, 32), "bfloat16 or float16"),
        (lambda: ctx.head_logits_q4(x.half(), x, x, 32), "uint8"),
        (lambda: ctx.head_logits_q4(x.half(), torch.zeros(4, 31, dtype=torch.uint8, device="cuda"), x, 32), "D / 2"),
        (lambda: ctx.head_logits_q4(x.half(), torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), x, 32), "scales"),
        (lambda: ctx.head_logits_q4(x.half(), torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), torch.zeros(4, 4, device="cuda"), 16),
         "group must be"),
        (lambda: ctx.head_logits_q4(x.half(), torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), torch.zeros(4, 2, device="cuda"), 32,
                                    zeros=torch.zeros(4, 2, device="cuda")), "zeros"),
        (lambda: ctx.head_logits_q4(x.half(), torch.zeros(4, 48, dtype=torch.uint8, device="cuda")[:, :32].flip(1), x, 32), "scales"),
    ]:
        with pytest.raises(V.VsmpError, match=words):
            call()
    torch.cuda.synchronize()
