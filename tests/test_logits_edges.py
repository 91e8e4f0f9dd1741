"""The operators around the pick at the ends of their domains, on the GPU."""
import numpy as np
import pytest

import verbo_amd as V
from helpers import log, mode_ctx
from test_logits_ops import check_adjusted, check_head, dev, pack, plain_adjust, plain_logprobs, q4_weights
from verbo_amd import decode

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


# ---- slots whose histories were trimmed ------------------------------------------------------------------


class Slots:
    """A decoder of slots beside its sequences' whole histories on the host."""

    def __init__(self, windows, n, cap=4096):
        self.n, self.said, self.windows = n, {}, dict(enumerate(windows))
        self.d = decode.BatchDecoder.with_slots(len(windows), n, cap=cap)

    def admit(self, slot, window, prompt):
        import torch

        self.windows[slot] = window
        self.said[slot] = [int(i) for i in prompt]
        self.d.admit(slot, V.Params(temp=0.0, repeat=1.0, repeat_last=window), prompt, torch.cuda.current_stream())

    def accept(self, live, ids):
        import torch

        self.d.accept_rows(dev(np.array(ids, np.int32)), dev(np.array(live, np.int32)), torch.ones(len(live), dtype=torch.int32, device="cuda"),
                           torch.cuda.current_stream())
        for s, t in zip(live, ids):
            self.said[s].append(int(t))

    def check(self, live, pens, prompts, rng):
        """Rows of the live slots against the whole histories' last window ids: the penalty's own window, at most the
        slot's repeat_last where that is above 0."""
        import torch

        x = rng.normal(0, 2, (len(live), self.n)).astype(np.float32)
        left = torch.empty(len(live), dtype=torch.int32, device="cuda")
        y = self.d.adjust_rows(dev(x), dev(np.array(live, np.int32)), V.to_device_penalties(pens),
                               prompt_len=dev(np.array(prompts, np.int32)) if prompts is not None else None, left=left)
        counted = []
        for s, p in zip(live, pens):
            w = self.windows[s]
            w = p.window if w <= 0 else w if p.window <= 0 else min(w, p.window)
            counted.append(V.Penalty(p.repeat, p.presence, p.frequency, w))
        want, tol = plain_adjust(x, counted, [self.said[s] for s in live], prompts)
        check_adjusted(y, left, want, tol)


def test_slots_windows_and_prompts_outlive_the_trims():
    """Histories that are cut from four windows to one again and again: what is penalised is always the last window
    ids, presence and frequency leave out the prompt however many of its ids are gone, and a slot's next sequence
    begins anew. Prompts shorter and longer than what a slot keeps; ids accepted on the device and from the host."""
    n = 40
    rng = np.random.default_rng(1)
    windows = [3, 5, 0, 2, 7]
    st = Slots(windows, n)
    lens = [4, 47, 30, 9, 0]
    for s, (w, k) in enumerate(zip(windows, lens)):
        st.admit(s, w, rng.integers(0, n, k).astype(np.int32))
    prompts = lens
    for step in range(70):
        live = [int(s) for s in rng.permutation(len(windows))[:rng.integers(1, len(windows) + 1)]]
        if step == 40:  # a new sequence in a slot that was trimmed before
            st.admit(0, 4, rng.integers(0, n, 6).astype(np.int32))
            prompts = [6] + lens[1:]
        if step == 50:  # ids from the host, past a trim
            ids = rng.integers(0, n, 23).astype(np.int32)
            st.d.accept_prompt(3, ids)
            st.said[3] += [int(i) for i in ids]
        pens = [V.Penalty(1.0 + 0.1 * s, 0.5, 0.25, int(rng.choice([0, -3, 1, 2, 4, 1000]))) for s in live]
        log("slots", step, live)
        st.check(live, pens, [prompts[s] for s in live], rng)
        st.check(live, pens, None, rng)
        st.accept(live, rng.integers(0, n, len(live)))


def test_slots_windows_in_a_replayed_graph():
    """A captured adjustment reads the slots as they are at each replay: after trims, and after a new sequence."""
    import torch

    n = 30
    rng = np.random.default_rng(2)
    st = Slots([2, 3], n)
    st.admit(0, 2, np.array([1, 2, 3], np.int32))
    st.admit(1, 3, np.array([4], np.int32))
    x = rng.normal(0, 2, (2, n)).astype(np.float32)
    xd, rows, prompt = dev(x), dev(np.array([1, 0], np.int32)), dev(np.array([1, 3], np.int32))
    pens = [V.Penalty(1.5, 1.0, 0.5, 0), V.Penalty(1.0, 2.0, 0.25, 0)]
    pd, out = V.to_device_penalties(pens), torch.empty(2, n, device="cuda")
    left = torch.empty(2, dtype=torch.int32, device="cuda")
    st.d.adjust_rows(xd, rows, pd, prompt_len=prompt, out=out, left=left)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        st.d.adjust_rows(xd, rows, pd, prompt_len=prompt, out=out, left=left)
    for step in range(30):
        if step == 17:
            st.admit(1, 3, np.array([7], np.int32))
        g.replay()
        counted = [V.Penalty(1.5, 1.0, 0.5, 3), V.Penalty(1.0, 2.0, 0.25, 2)]
        check_adjusted(out, left, *plain_adjust(x, counted, [st.said[1], st.said[0]], [1, 3]))
        st.accept([0, 1], rng.integers(0, n, 2))


def test_serve_leaves_the_prompt_out():
    """Requests whose presence and frequency penalties leave their prompts out, and ones whose penalties count them,
    over windows that are cut several times: greedy picks over constant logits, by the rules alone."""
    import torch

    n = 24
    base = np.linspace(6.0, 0.0, n).astype(np.float32)
    cases = [  # prompt, window, penalty, prompt_len, ids to generate, arrival
        ([0, 1, 2, 3, 0, 1], 3, V.Penalty(presence=1.0, frequency=0.75), 6, 40, 0),
        ([0, 1, 2, 3, 0, 1], 3, V.Penalty(presence=1.0, frequency=0.75), 0, 40, 0),
        ([5, 0, 0], 4, V.Penalty(frequency=0.5), 3, 30, 2),
        ([5, 0, 0, 7], 4, V.Penalty(repeat=1.5, frequency=0.5, window=2), 2, 30, 3),
        (list(range(20)), 2, V.Penalty(presence=3.0), 20, 25, 4),
        ([0, 1, 2], 0, V.Penalty(presence=2.0), 3, 20, 5),
    ]
    reqs = [decode.Request(p, decode.Opts(max_tokens=m, temp=0.0), repeat_last=w, arrival=at, penalty=pen, prompt_len=k)
            for p, w, pen, k, m, at in cases]
    d = decode.BatchDecoder.with_slots(3, n)
    res = d.serve(reqs, lambda js, steps, last: torch.from_numpy(np.tile(base, (len(js), 1))).cuda())
    for (prompt, w, pen, k, m, _), (toks, _) in zip(cases, res):
        said = list(prompt)
        win = pen.window if w <= 0 else w if pen.window <= 0 else min(w, pen.window)
        for _ in range(m):
            y, _ = plain_adjust(base[None], [V.Penalty(pen.repeat, pen.presence, pen.frequency, win)], [said], [k])
            said.append(int(y[0].argmax()))
        assert toks == said[len(prompt):], (prompt, w, k)
    assert res[0][0] != res[1][0]


def test_serve_uploads_penalties_when_the_live_requests_change(monkeypatch):
    """Penalties go to the device once for as long as the same requests are live in the same slots."""
    import torch

    n, calls = 12, []
    upload = decode.to_device_penalties
    monkeypatch.setattr(decode, "to_device_penalties", lambda p, dev: calls.append(len(p)) or upload(p, dev))
    reqs = [decode.Request([0], decode.Opts(max_tokens=m, temp=0.0), repeat_last=0, arrival=at, penalty=V.Penalty(presence=9.0))
            for m, at in ((9, 0), (4, 2), (6, 3))]
    d = decode.BatchDecoder.with_slots(2, n)
    base = torch.linspace(3.0, 0.0, n, device="cuda")
    res = d.serve(reqs, lambda js, steps, last: base.expand(len(js), n).contiguous())
    assert [t for t, _ in res] == [list(range(1, m + 1)) for m in (9, 4, 6)]
    # request 0 alone, with 1 until its slot is free, with 2, 2 alone
    assert calls == [1, 2, 2, 1]


# ---- scratch, arguments, streams -----------------------------------------------------------------------------


@pytest.mark.parametrize("warm", [(2, 500), (2000, 20000)])
def test_any_first_call_holds_the_scratch(warm):
    """After one call of vsmp_logprobs, whether it cut its rows into parts or not, calls of every shape are captured."""
    import torch

    fresh = V.Context(0)
    fresh.logprobs(torch.randn(*warm, device="cuda"), torch.zeros(warm[0], 1, dtype=torch.int32, device="cuda"))
    x, ids = torch.randn(2, 50000, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        got = fresh.logprobs(x, ids)
    for _ in range(3):
        x.normal_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, fresh.logprobs(x, ids)):
            assert torch.equal(a, b)


def test_an_empty_mask_table_is_refused(ctx):
    """A table without masks is no way to say that rows are not masked."""
    import torch

    x = torch.zeros(2, 64, device="cuda")
    none = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(mask_row=torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(V.VsmpError, match="mask"):
            ctx.adjust_logits(x, mask=none, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_adjusted_rows_between_the_logits(ctx, dtype):
    """Logits and output in one buffer, row by row in turn, share no byte."""
    import torch

    B, n = 5, 6001
    rng = np.random.default_rng(7)
    x = dev(rng.normal(0, 3, (B, n)).astype(np.float32), dtype)
    step = 4 * (2 * n + 3)  # bytes from a row to the next
    buf = torch.zeros(B * step, dtype=torch.uint8, device="cuda").view(B, step)
    size = x.element_size()
    src = buf[:, :n * size].view(x.dtype)
    src.copy_(x)
    out = buf[:, 4 * (n + 1):4 * (2 * n + 1)].view(torch.float32)
    bias = dict(bias_ids=dev(np.arange(B, dtype=np.int32)), bias=torch.ones(B, device="cuda"), bias_off=dev(np.arange(B + 1, dtype=np.int32)))
    got = ctx.adjust_logits(src, out=out, **bias)
    assert got is out and torch.equal(got, ctx.adjust_logits(x, **bias)) and torch.equal(src, x)


def test_outputs_belong_to_the_callers_stream(ctx):
    """A call on a stream of its own does not take memory that the current stream may still be using, and what it
    returns is not handed to that stream again while the current one may be using it."""
    import torch

    B, n, D = 64, 40000, 256
    x = torch.randn(B, n, device="cuda")
    half = x.bfloat16()
    ids = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    q, s, z, _ = q4_weights(1, n, D, 64)
    hidden = torch.randn(B, D, device="cuda").bfloat16()
    d = decode.BatchDecoder.with_slots(B, n)
    rows = torch.arange(B, dtype=torch.int32, device="cuda")
    head = torch.randn(n, D, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    calls = [lambda st: ctx.adjust_logits(half, stream=st), lambda st: d.adjust_rows(half, rows, stream=st),
             lambda st: ctx.head_logits_q4(hidden, q, s, 64, stream=st), lambda st: ctx.head_logits(hidden, head, stream=st)]
    for call in calls:
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        want = call(None)  # the context's scratch is there from here on
        torch.cuda.synchronize()
        old = torch.empty(B, n, device="cuda")
        at = old.data_ptr()
        del old  # free for the current stream alone
        got = call(side)
        assert got.data_ptr() != at
        side.synchronize()
        assert torch.equal(got, want)
        torch.cuda._sleep(400_000_000)  # the current stream is busy with `got`
        keep, used = got + 0.0, torch.cuda.Event()
        used.record()
        at = got.data_ptr()
        del got
        with torch.cuda.stream(side):
            again = torch.empty(B, n, device="cuda")
        assert again.data_ptr() != at or used.query()  # free again only once the current stream has read it
        again.fill_(7.0)
        torch.cuda.synchronize()
        assert torch.equal(keep, want)
        del again, keep, want
    for call in (lambda st: ctx.logprobs(x, ids, stream=st), lambda st: (ctx.pick_batch(x, V.Params(temp=0.0), stream=st),)):
        call(None)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        old = [torch.empty(B, device="cuda") for _ in range(16)]
        at = [t.data_ptr() for t in old]
        del old
        assert not {t.data_ptr() for t in call(side)} & set(at)
        torch.cuda.synchronize()


# ---- the head with 4-bit weights ---------------------------------------------------------------------------


@pytest.mark.parametrize("G,zeros,scales,dtype", [(32, True, "f32", "bf16"), (64, False, "bf16", "f16"), (128, True, "f16", "bf16")])
def test_head_q4_every_small_hidden_size(ctx, G, zeros, scales, dtype):
    """Every hidden size below 256, which is staged whole, with batches around 16 rows."""
    rng = np.random.default_rng(G)
    for D in range(G, 256, G):
        q, s, z, w = q4_weights(D, 131, D, G, scales, zeros)
        for B in (1, 15, 16, 17, 33):
            hidden = dev(rng.normal(0, 1, (B, D)).astype(np.float32), dtype)
            log("small head", G, D, B)
            check_head(ctx.head_logits_q4(hidden, q, s, G, zeros=z), hidden, s, z, w, G)


# ---- far operands --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("D,scales", [(64, "f32"), (640, "f32"), (640, "bf16")])
def test_head_q4_operands_far_apart(ctx, D, scales):
    """Hidden rows 2^30 elements apart, and columns of the weights, scales and zero points as far apart as they may
    be: column and row offsets beyond 2^32 bytes."""
    import torch

    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of device memory")
    n, G = 300, 32
    q, s, z, w = q4_weights(D, n, D, G, scales, True)

    def far(t, ld):
        rows, cols = t.shape
        v = torch.empty((rows - 1) * ld + cols, dtype=t.dtype, device="cuda").as_strided((rows, cols), (ld, 1))
        v.copy_(t)
        return v

    fq, fs, fz = far(q, (1 << 26) - 16), far(s, (1 << 24) - 1), far(z, (1 << 26) - 1)
    for B in (3, 9, 70):
        hidden = torch.randn(B, D, device="cuda").bfloat16()
        log("far head", D, B)
        fh = far(hidden, 1 << 30) if B < 70 else hidden
        got = ctx.head_logits_q4(fh, fq, fs, G, zeros=fz)
        check_head(got, hidden, s, z, w, G)
        assert torch.equal(got, ctx.head_logits_q4(hidden, q, s, G, zeros=z))
        del fh


def test_masks_far_apart(ctx):
    """A table whose masks lie 2^30 words apart."""
    import torch

    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    n, ld = 5000, 1 << 30
    rng = np.random.default_rng(5)
    allow = [rng.random(n) < 0.5 for _ in range(4)]
    near = dev(pack(allow, n, (n + 31) // 32))
    table = torch.empty(3 * ld + near.shape[1], dtype=torch.int32, device="cuda").as_strided(near.shape, (ld, 1))
    table.copy_(near)
    x = torch.randn(6, n, device="cuda")
    row = dev(np.array([3, -1, 0, 2, 3, 1], np.int32))
    assert torch.equal(ctx.adjust_logits(x, mask=table, mask_row=row), ctx.adjust_logits(x, mask=near, mask_row=row))
    assert torch.equal(ctx.adjust_logits(x[:4], mask=table), ctx.adjust_logits(x[:4], mask=near))


# ---- the largest sizes, the smallest values ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_largest_vocabulary(ctx, dtype):
    """Rows of 2^20 logits: adjusted, and their log-probabilities and ranks."""
    import torch

    n, B = 1 << 20, 2
    rng = np.random.default_rng(3)
    x = rng.normal(0, 3, (B, n)).astype(np.float32)
    xd = dev(x, dtype)
    xs = xd.float().cpu().numpy()
    hists = [rng.integers(0, n, 5000), np.array([0, n - 1, n - 1, 77])]
    flat, off = np.concatenate(hists).astype(np.int32), np.array([0, 5000, 5004], np.int32)
    masks = [None, rng.random(n) < 0.5]
    left = torch.empty(B, dtype=torch.int32, device="cuda")
    pen = V.Penalty(1.25, 0.5, 0.25, 4000)
    log("largest", dtype)
    y = ctx.adjust_logits(xd, pen, dev(flat), dev(off), mask=dev(pack(masks[1:], n, n // 32)), mask_row=dev(np.array([-1, 0], np.int32)),
                          left=left)
    check_adjusted(y, left, *plain_adjust(xs, [pen], hists, None, None, masks))
    ids = np.concatenate([np.argsort(-xs, 1, kind="stable")[:, :4], np.tile([0, n - 1, n, n // 2], (B, 1))], 1).astype(np.int32)
    lp, rank, lse = ctx.logprobs(xd, dev(ids))
    wl, _, wz, tol = plain_logprobs(xs, ids)
    assert np.array_equal(rank.cpu().numpy(), plain_ranks(xs, ids))
    assert (np.abs(lse.cpu().numpy() - wz) <= tol + 2.0 ** -24 * np.abs(wz)).all()
    g, fin = lp.cpu().numpy(), np.isfinite(wl)
    # the bound of the sums, and a rounding each of the difference from the largest logit and of the result
    with np.errstate(invalid="ignore"):
        most = tol[:, None] + 2.0 ** -24 * (4 * np.abs(wl) + tol[:, None])
        assert (np.abs(g - wl) <= most)[fin].all() and np.array_equal(g[~fin], wl[~fin])


@pytest.mark.parametrize("D", [64, 256])
def test_head_q4_the_largest_vocabulary(ctx, D):
    n, G = 1 << 20, 64
    import torch

    q, s, z, w = q4_weights(D, n, D, G, "bf16", True)
    hidden = torch.randn(2, D, device="cuda").bfloat16()
    got = ctx.head_logits_q4(hidden, q, s, G, zeros=z)
    check_head(got, hidden, s, z, w, G)


def test_denormal_logits(ctx):
    """Logits and adjusted values below the smallest normal float keep their bits, order and ties."""
    n = 5000
    rng = np.random.default_rng(9)
    x = (rng.integers(-40, 41, (3, n)) * np.float32(2.0 ** -149)).astype(np.float32)
    x[1] = rng.integers(-3, 4, n).astype(np.float32) * np.float32(2.0 ** -126)
    x[2, ::7] = -0.0
    ids = np.concatenate([rng.integers(0, n, (3, 50)), np.argsort(-x, 1, kind="stable")[:, :8]], 1).astype(np.int32)
    lp, rank, lse = ctx.logprobs(dev(x), dev(ids))
    assert np.array_equal(rank.cpu().numpy(), plain_ranks(x, ids))
    h, off = rng.integers(0, n, 9000).astype(np.int32), np.array([0, 3000, 6000, 9000], np.int32)
    got = ctx.adjust_logits(dev(x), V.Penalty(repeat=1.5), dev(h), dev(off)).cpu().numpy()
    want = x.copy()
    for r in range(3):
        s = np.unique(h[off[r]:off[r + 1]])
        want[r, s] = np.where(x[r, s] > 0, x[r, s] / np.float32(1.5), x[r, s] * np.float32(1.5))
    assert np.array_equal(got.view(np.int32), want.view(np.int32))


@pytest.mark.parametrize("D,B", [(96, 5), (640, 3), (640, 9), (640, 30), (640, 64)])
def test_head_q4_rows_do_not_touch_each_other(ctx, D, B):
    """A row of NaN (the documentation asks for finite hidden states) leaves the other rows' bits alone."""
    import torch

    q, s, z, _ = q4_weights(D, 333, D, 32, "f32", True)
    hidden = torch.randn(B, D, device="cuda").bfloat16()
    want = ctx.head_logits_q4(hidden, q, s, 32, zeros=z)
    hidden[B // 2] = NAN
    got = ctx.head_logits_q4(hidden, q, s, 32, zeros=z)
    rest = [r for r in range(B) if r != B // 2]
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[B // 2]).all()


def test_every_slot_without_a_slot_list():
    """vsmp_bsampler_adjust_rows with rows NULL: row i is slot i, for more slots than one launch counts."""
    import torch

    n, slots = 7, 9001
    rng = np.random.default_rng(4)
    d = decode.BatchDecoder([decode.Opts(temp=0.0)] * slots, n, repeat_last=1, cap=4)
    said = []
    live = torch.ones(slots, dtype=torch.int32, device="cuda")
    for _ in range(7):
        said.append(rng.integers(0, n, slots).astype(np.int32))
        d.accept(dev(said[-1]), live, torch.cuda.current_stream())
    x = rng.normal(0, 2, (slots, n)).astype(np.float32)
    xd, out, left = dev(x), torch.empty(slots, n, device="cuda"), torch.empty(slots, dtype=torch.int32, device="cuda")
    pens = V.to_device_penalties(np.array([(1.0, 0.5, 0.25, 0)] * slots, V.PENALTY_DTYPE))
    prompt = torch.from_numpy((np.arange(slots) % 9).astype(np.int32)).cuda()
    rc = d.lib.vsmp_bsampler_adjust_rows(d._h, xd.data_ptr(), 0, n, n, None, slots, pens.data_ptr(), 1, prompt.data_ptr(), None, None,
                                         None, None, 0, 0, None, out.data_ptr(), n, left.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    want = x.copy()
    rows = np.where(np.arange(slots) % 9 < 7)[0]  # the last id is not the prompt's
    want[rows, said[-1][rows]] -= np.float32(0.75)
    assert np.array_equal(out.cpu().numpy(), want) and (left == n).all()


def test_a_stream_is_known_by_its_address(ctx):
    """Every call takes any object that has a stream's address, whether it allocates its output or not."""
    import types

    import torch

    x, ids = torch.randn(3, 5000, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    bare = types.SimpleNamespace(cuda_stream=side.cuda_stream)
    calls = [lambda st: ctx.adjust_logits(x, stream=st), lambda st: ctx.logprobs(x, ids, stream=st)[0],
             lambda st: ctx.pick_batch(x[:, :5000], V.Params(temp=0.0), stream=st)]
    for call in calls:
        want = call(None)
        torch.cuda.synchronize()
        for st in (bare, side, torch.cuda.default_stream(), torch.cuda.current_stream()):
            got = call(st)
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_serve_follows_a_penalty_that_changes():
    """A request's penalty and prompt length changed between steps, in place or replaced, hold from the next pick on."""
    import torch

    n = 12
    base = torch.linspace(3.0, 0.0, n, device="cuda")
    req = decode.Request([0], decode.Opts(max_tokens=6, temp=0.0), repeat_last=0, penalty=V.Penalty(presence=9.0))

    def logits(js, steps, last):
        if steps[0] == 2:
            req.penalty.presence = 0.0
        if steps[0] == 4:
            req.penalty = V.Penalty(presence=9.0)
        if steps[0] == 5:
            req.prompt_len = 1
        return base.expand(1, n).contiguous()

    toks, _ = decode.BatchDecoder.with_slots(1, n).serve([req], logits)[0]
    # 0 is the prompt; 1 and 2 penalised apart from it; nothing penalised; 0, 1 and 2 penalised; 0 said by itself too
    assert toks == [1, 2, 0, 0, 3, 4]
