"""Selection where masks are finite numbers and logits are large, and steps of a cache whose rows ask for more pages
than 32 bits count, on the GPU.

Tolerances count roundings: u = 2^-24 is the most that rounding to fp32 takes, relative to the value."""
import numpy as np
import pytest

import verbo_amd as V
from helpers import log, mode_ctx
from test_search_ops import INF, U, continuations, i32, torch_type

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch

    assert torch.cuda.is_available(), "the gpu tests need a ROCm device"
    return mode_ctx()


# ---- selection: finite masks, large logits ---------------------------------------------------------------


def lse_tolerance(vocab, dtype):
    """How far a row's log of a sum may be off. Terms at most 40 below the largest (others count for less than e^-40 each)
    have arguments that are rounded twice on the way from the term to the row's maximum, each time by 40 u at most,
    and log2 e is off by a quarter of a rounding (10 u): 90 u whatever the number of maxima on the way. An exponential is
    off by 2 u, what makes good the argument's rounding by 3 u. A thread adds a step of 16 logits (32 of 2 bytes)
    one by one, then the steps, each with a factor for the new maximum (an exponential and a product, 3 u); the same factor
    comes in three joins; a wave adds in 6 turns, what is beyond is in 64 bits. A row's end is one step more."""
    per = 16 if dtype == "f32" else 32
    steps = -(-vocab // (256 * per)) + 1
    return (90 + 5 + per + 4 * steps + 9 + 6) * U


def check(ctx, x, scores, n, dtype, stops=()):
    """The step on device rows x against the definition in 64 bits, in which logits of size M leave lse and x - lse with
    2^-53 M each, here and there. Where two neighbours in the order lie closer than the tolerance either may come first."""
    import torch

    G, W = scores.shape
    r = V.BeamStep(*[t.cpu().numpy() for t in ctx.beam_select(x, torch.from_numpy(scores).cuda(), n, stop_ids=stops)])
    host = x.double().cpu().numpy()
    vocab = host.shape[1]
    for g, (s, row, v, tok) in enumerate(continuations(host, scores, W)):
        rows = host[g * W:(g + 1) * W]
        tops = np.where(np.isnan(rows), -INF, rows).max(1)
        big = np.abs(tops[np.isfinite(tops)]).max(initial=0.0)
        tol = lse_tolerance(vocab, dtype) + 4 * 2.0 ** -53 * big
        end = np.isin(tok, list(stops))
        place = {(int(a), int(t)): k for k, (a, t) in enumerate(zip(row, tok))}
        go = np.flatnonzero(~end)[:n]
        assert (r.token[g] >= 0).sum() == go.size, (g, r.token[g], go.size)
        for i in range(go.size):
            k = place[(int(r.parent[g, i]), int(r.token[g, i]))]
            # (a score that lies far below has the roundings of its own size)
            near = tol + 4 * 2.0 ** -53 * abs(s[k])
            assert not end[k] and abs(float(r.score[g, i]) - s[k]) <= near + U * abs(s[k]), (g, i, r.score[g, i], s[k])
            if k != go[i]:
                assert abs(s[k] - s[go[i]]) <= 2 * near and row[k] != row[go[i]], (g, i, s[k], s[go[i]])
    return r


SHAPES = [  # G, W, n, vocab: a wave's end; four waves'; several parts; many parts
    (2, 3, 4, 5003),
    (2, 9, 20, 9001),
    (1, 2, 5, 70001),
]


@pytest.mark.parametrize("mask,dtype", [(m, d) for d in ("f32", "bf16") for m in (-1e4, -1e6, -1e8, -1e9, -1e10, -1e15, -1e20, -1e30, -1e38)] +
                         [(-1e4, "f16"), (-6e4, "f16")])
@pytest.mark.parametrize("left", ["half", "a part", "few", "one", "one behind the last whole group", "none"])
def test_select_finite_masks(ctx, mask, dtype, left):
    """Rows masked with a finite number: whole lanes and whole parts of it, all but some tokens, and all."""
    import torch

    log("finite mask", mask, dtype, left)
    for G, W, n, vocab in SHAPES:
        rng = np.random.default_rng(vocab + W)
        x = rng.normal(0, 3, (G * W, vocab)).astype(np.float32)
        keep = np.zeros(x.shape, bool)
        if left == "half":
            keep[:, vocab // 2:] = True
        elif left == "a part":
            keep[:, 4096:4200] = True
        elif left == "few":
            keep[np.arange(G * W)[:, None], rng.integers(0, vocab, (G * W, 7))] = True
        elif left == "one":
            keep[np.arange(G * W), rng.integers(0, vocab, G * W)] = True
        elif left != "none":
            keep[:, -1] = True
        x = torch.from_numpy(np.where(keep, x, np.float32(mask))).cuda().to(torch_type(dtype))
        scores = -rng.uniform(1, 5, (G, W)).astype(np.float32)
        check(ctx, x, scores, n, dtype, [vocab - 2, 4100])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [1e4, 11356.0, 11357.0, 1.2e4, 1e5, 1e6, 1e8, 1e15, 1e20, 1e30, 3e38])
def test_select_large_logits(ctx, shift, dtype):
    """Rows that are large throughout, in either sign, on both sides of what the kernel's shorter exponential serves."""
    import torch

    log("large logits", shift, dtype)
    for G, W, n, vocab in SHAPES:
        rng = np.random.default_rng(vocab)
        x = rng.normal(0, 3, (G * W, vocab)).astype(np.float32)
        with np.errstate(over="ignore"):
            x += np.where(np.arange(G * W)[:, None] % 2 == 0, shift, -shift).astype(np.float32)
        x = torch.from_numpy(x).cuda().to(torch_type(dtype))
        check(ctx, x, -rng.uniform(1, 5, (G, W)).astype(np.float32), n, dtype, [3])


def test_select_mixed_masks_in_many_rows(ctx):
    """A part a row (more rows than workgroups of four a CU): every row with a mask of its own."""
    import torch

    log("mixed masks")
    G, W, n, vocab = 150, 8, 8, 4999
    rng = np.random.default_rng(2)
    masks = np.array([-1e4, -1e9, -1e10, -1e30, -1e38, -3e38, -INF, 0.0], np.float32)[rng.integers(0, 8, G * W)]
    x = rng.normal(0, 3, (G * W, vocab)).astype(np.float32)
    x = np.where(rng.random(x.shape) < 0.01, x, masks[:, None])
    check(ctx, torch.from_numpy(x).cuda(), -rng.uniform(1, 5, (G, W)).astype(np.float32), n, "f32", [7])


# ---- a cache in pages ------------------------------------------------------------------------------------


def test_pages_rows_that_together_ask_for_more_than_32_bits_count(ctx):
    """1,024 rows that ask for 2^21 pages each and more: rows that fit get their pages, all others none."""
    import torch

    P, R, cap = 1000, 1024, (1 << 21) + 8192
    start = V.Pages.empty(1, 1, P, 1)
    to = V.Pages(torch.empty(R, cap, dtype=torch.int32, device="cuda"), i32(np.zeros(R)), i32(np.zeros(P)), 1)
    want = np.full(R, cap)
    want[:2] = 5, 7
    assert int(want.sum()) >= 1 << 31
    log("more than 32 bits count")
    got, ok = ctx.pages_step(start, i32(np.full(R, -1)), i32(want), out=to)
    fits = np.cumsum(want) <= P
    assert ok.cpu().numpy().tolist() == fits.astype(int).tolist()
    assert got.lens.cpu().numpy().tolist() == np.where(fits, want, 0).tolist()
    assert got.ref.cpu().numpy().tolist() == [1] * 12 + [0] * (P - 12)
    assert got.table[0, :5].tolist() == [0, 1, 2, 3, 4] and got.table[1, :7].tolist() == [5, 6, 7, 8, 9, 10, 11]
    assert int((got.table >= 0).sum()) == 12


@pytest.mark.parametrize("rows,n_pages", [(6, 40), (64, 100), (200, 300), (6, 65537), (1025, 300)])
def test_pages_that_a_row_asked_for_in_vain_count(ctx, rows, n_pages):
    """Behind a row that the pool has too few pages for, rows that need a page get none, and rows that need none, or are cut,
    go on; a row that the table has too little room for asks for none."""
    cap, T = n_pages + 8, 2
    table = np.full((rows, cap), -1, np.int32)
    table[:, 0] = np.arange(rows) % n_pages  # where there are more rows than pages they share them
    start = V.Pages(i32(table), i32(np.full(rows, 1)), i32(np.bincount(table[:, 0], minlength=n_pages)), T)
    add = np.zeros(rows, int)
    add[:6] = 2 * cap, n_pages * T if rows < n_pages else 0, 2, 1, 0, -1
    log("asked for in vain", rows, n_pages)
    to, ok = ctx.pages_step(start, add=i32(add))
    m = [0, 0, 0, 1, 1, 1] if rows < n_pages else [0, 1, 0, 0, 1, 1]
    assert ok.cpu().numpy()[:6].tolist() == m and bool(ok[6:].all())
    assert to.lens.cpu().numpy()[:6].tolist() == [1 + int(a) * o for a, o in zip(add, m)]


# ---- streams ---------------------------------------------------------------------------------------------


def test_outputs_of_calls_on_the_default_stream_are_its_memory(ctx):
    """From within another stream: once freed, the default stream's next tensor of that size takes the memory, and the
    other stream's does not."""
    import torch

    G, n = 200_003, 8
    x, scores = torch.randn(G, 9, device="cuda"), torch.full((G, 1), -1.0, device="cuda")
    want = ctx.beam_select(x, scores, n)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    log("default stream")
    with torch.cuda.stream(torch.cuda.Stream()):
        got = ctx.beam_select(x, scores, n, stream=torch.cuda.default_stream())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        at = got.token.data_ptr()
        del got
        other = torch.empty(6, G, n, dtype=torch.int32, device="cuda")
    again = torch.empty(6, G, n, dtype=torch.int32, device="cuda")
    assert other.data_ptr() != at and again.data_ptr() == at


@pytest.mark.parametrize("call", ["reorder", "step", "compact"])
@pytest.mark.parametrize("how", ["argument", "current"])
def test_planes_that_are_gone_before_their_call_has_run(ctx, call, how):
    """Planes made on one stream and dropped after a call on another, which is busy: what is allocated then does not take
    the addresses' memory, and the call finds them."""
    import torch

    st = torch.cuda.Stream()
    a = torch.randn(4096, 4096, device="cuda")
    x = torch.arange(4 * 6, dtype=torch.int32, device="cuda").view(4, 6, 1)
    parent = i32([1, 1, 3, 2])
    pages = V.Pages(i32([[3, -1], [3, 1]]), i32([3, 8]), i32([0, 1, 0, 2]), 6)
    want = {"reorder": lambda: ctx.reorder_rows(V.Planes([x.clone()], token_dim=1), parent, 2),
            "step": lambda: ctx.pages_step(pages, add=1, cache=V.Planes([x.clone()], token_dim=1))[0].table,
            "compact": lambda: ctx.pages_compact(pages, cache=V.Planes([x.clone()], token_dim=1))[0].table}[call]()
    planes = V.Planes([x], token_dim=1)
    at = planes._ptrs.data_ptr()
    log("gone", call, how)
    b = a @ a
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(100):
            torch.mm(a, a, out=b)
    if how == "current":
        with torch.cuda.stream(st):
            got = ctx.reorder_rows(planes, parent, 2) if call == "reorder" else \
                (ctx.pages_step(pages, add=1, cache=planes) if call == "step" else ctx.pages_compact(pages, cache=planes))[0]
    else:
        got = ctx.reorder_rows(planes, parent, 2, stream=st) if call == "reorder" else \
            (ctx.pages_step(pages, add=1, cache=planes, stream=st) if call == "step" else ctx.pages_compact(pages, cache=planes, stream=st))[0]
    del planes
    new = [torch.empty(1, dtype=torch.int64, device="cuda") for _ in range(100)]
    busy = not st.query()
    torch.cuda.synchronize()
    assert busy and at not in [t.data_ptr() for t in new]
    rows = x.view(4, 6).tolist()
    was = np.arange(24).reshape(4, 6).tolist()
    if call == "reorder":
        assert rows == [was[k] for k in (1, 1, 3, 2)]
    else:
        assert torch.equal(got.table, want)
        if call == "step":    # row 0 shares its begun page with a full one of row 1: it copies three tokens to page 0
            assert rows == [was[3][:3] + was[0][3:]] + was[1:]
        else:                 # pages 1 and 3 move to 1 and 0
            assert rows == [was[3]] + was[1:]


# ---- numbers that a C int does not hold ------------------------------------------------------------------


def test_numbers_beyond_32_bits(ctx):
    """Refused, or, as stop tokens, outside the vocabulary: cut to 32 bits each of these would be a number that serves."""
    import torch

    x, scores = torch.zeros(4, 10, device="cuda"), torch.zeros(2, 2, device="cuda")
    x[:, 3] = 5.0
    log("numbers beyond 32 bits")
    assert ctx.beam_select(x, scores, stop_ids=[(1 << 32) + 3, -(1 << 32) + 3, 1 << 40]).n_end.tolist() == [0, 0]
    state = torch.zeros(4, 6, dtype=torch.int32, device="cuda")
    parent, pages = i32([1, 0, 2, 3]), V.Pages.empty(4, 4, 16, 4)
    wide = torch.empty(2, (1 << 30) + 16, device="cuda")  # rows of 2^32 + 64 bytes
    for make in (lambda: ctx.beam_select(x, scores, (1 << 32) + 2), lambda: ctx.reorder_rows(V.Planes([state]), parent, (1 << 32) + 2),
                 lambda: V.Planes([wide]), lambda: V.Planes([wide.view(torch.uint8)]),
                 lambda: V.Pages(pages.table, pages.lens, pages.ref, (1 << 32) + 4), lambda: ctx.pages_step(pages, add=1 << 31),
                 lambda: ctx.pages_step(pages, add=(1 << 32) + 1), lambda: ctx.pages_step(pages, add=-(1 << 31) - 1)):
        with pytest.raises(V.VsmpError, match="32 bits"):
            make()
    with pytest.raises(V.VsmpError):
        V.Planes([wide.view(torch.uint8).view(2, -1, 1)], token_dim=1)
    to, ok = ctx.pages_step(pages, add=(1 << 31) - 1)
    assert ok.tolist() == [0] * 4 and to.lens.tolist() == [0] * 4
