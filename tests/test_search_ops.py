"""Beams and the states behind them on the GPU (include/vsmp_beam.h): the selection of a step against its definition in 64
bits, rows of states against indexing, a cache in pages against a model of it that holds every row's tokens, at the
sizes, masks, strides and shortages where they can go wrong; then together, from replayed graphs and on other streams.

Tolerances count roundings: u = 2^-24 is the most that rounding to fp32 takes, relative to the value."""
import numpy as np
import pytest

import verbo_amd as V
from helpers import log, mode_ctx

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


@pytest.fixture(scope="module")
def ctx():
    import torch

    assert torch.cuda.is_available(), "the gpu tests need a ROCm device"
    return mode_ctx()


def torch_type(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8, "i32": torch.int32}[name]


def i32(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


# ---- the selection ---------------------------------------------------------------------------------------


def continuations(x, scores, W):
    """For each group its continuations in order: (s, row, x, token); x float64 rows."""
    out = []
    for g in range(len(scores)):
        found = []
        for b in range(W):
            v, sc = x[g * W + b], float(scores[g][b])
            with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                top = v.max()
                lse = top + np.log(np.exp(v - top).sum())
            if not np.isfinite(sc) or not np.isfinite(lse):
                continue
            t = np.flatnonzero(v > -INF)
            found.append(np.stack([-(sc + (v[t] - lse)), np.full(t.size, b, float), -v[t], t.astype(float)], 1))
        f = np.concatenate(found) if found else np.zeros((0, 4))
        f = f[np.lexsort((f[:, 3], f[:, 2], f[:, 1], f[:, 0]))]
        out.append((-f[:, 0], g * W + f[:, 1].astype(int), -f[:, 2], f[:, 3].astype(int)))
    return out


# Of the log of a sum: terms at most 40 below the largest (others count for nothing) have exponents off by 40 * 2 roundings
# and an exponential off by 2; a thread adds at most 2^20 / 256 of them, and their sums join in 64 bits.
LSE = (2 * 40 + 2 + 4096) * U


def check_select(ctx, x, scores, n, stops=(), got=None):
    """The step on device rows x against the definition. Where two neighbours in the order lie closer than the
    sums' tolerance, either may come first: the score that the definition gives what was returned decides."""
    G, W = scores.shape
    import torch

    r = ctx.beam_select(x, torch.from_numpy(scores).cuda(), n, stop_ids=stops) if got is None else got
    r = V.BeamStep(*[t.cpu().numpy() for t in r])
    host = x.double().cpu().numpy()
    for g, (s, row, v, tok) in enumerate(continuations(host, scores, W)):
        end = np.isin(tok, [t for t in stops])
        early = np.arange(s.size) < n
        place = {(int(a), int(t)): k for k, (a, t) in enumerate(zip(row, tok))}
        for sel, names in ((np.flatnonzero(~end)[:n], ("token", "parent", "score")), (np.flatnonzero(end & early), ("end_token", "end_parent", "end_score"))):
            a, b, c = (getattr(r, k)[g] for k in names)
            close = np.abs(np.diff(s[:n + 1])).min(initial=INF) < 2 * LSE
            if names[0] == "end_token" and not close:
                assert r.n_end[g] == sel.size, (g, r.n_end[g], sel.size)
            m = sel.size if names[0] == "token" else int(r.n_end[g])
            for i in range(n):
                if i >= m:
                    assert (a[i], b[i], c[i]) == (-1, g * W + i % W, -INF), (g, i, a[i], b[i], c[i])
                    continue
                k = place[(int(b[i]), int(a[i]))]
                assert end[k] == (names[0] == "end_token")
                if i < sel.size and k != sel[i]:
                    assert abs(s[k] - s[sel[i]]) <= 2 * LSE and (b[i] != row[sel[i]]), (g, i, names, a[i], b[i], s[k], s[sel[i]])
                assert abs(c[i] - s[k]) <= LSE + U * abs(s[k]), (g, i, c[i], s[k])
    return r


def logits(rng, B, vocab, dtype, ld=None, shift=0):
    import torch

    x = rng.normal(0, 2, (B, vocab)).astype(np.float32)
    x[:, rng.integers(0, vocab, 5)] += rng.uniform(2, 8, (B, 5)).astype(np.float32)
    ld = ld or vocab
    buf = torch.full((shift + B * ld,), 1e4, dtype=torch_type(dtype), device="cuda")  # what lies between rows would win
    v = buf[shift:shift + B * ld].view(B, ld)[:, :vocab]
    v.copy_(torch.from_numpy(x).cuda())
    return v


@pytest.mark.parametrize("G,W,n,vocab,dtype,pad,shift,stops", [
    (1, 1, 1, 1, "f32", 0, 0, 0),
    (1, 1, 4, 2, "bf16", 0, 0, 1),
    (3, 2, 5, 7, "f16", 3, 1, 2),
    (2, 3, 3, 63, "f32", 1, 1, 0),
    (5, 4, 4, 257, "bf16", 1, 3, 3),
    (2, 64, 64, 300, "f32", 0, 0, 4),
    (3, 64, 1, 1025, "f16", 7, 5, 1),
    (4, 1, 64, 4097, "f32", 0, 0, 2),
    (1, 8, 8, 4096, "bf16", 0, 0, 16),
    (2, 7, 9, 8193, "f16", 2, 1, 1),
    (1, 4, 4, 49152, "f32", 0, 0, 1),
    (24, 5, 5, 50257, "f16", 0, 0, 3),
    (16, 1, 8, 151936, "bf16", 0, 0, 1),
    (33, 6, 7, 32001, "bf16", 3, 1, 2),
    (1, 3, 5, 262147, "f32", 1, 1, 0),
    (1, 1, 2, 1 << 20, "f16", 0, 0, 1),
    (700, 8, 2, 1003, "f32", 0, 0, 1),   # more parts than one launch holds
    (70, 64, 3, 513, "bf16", 0, 0, 0),
])
def test_select(ctx, G, W, n, vocab, dtype, pad, shift, stops):
    log("select", G, W, n, vocab, dtype)
    rng = np.random.default_rng(G * 1000 + W * 100 + n + vocab)
    x = logits(rng, G * W, vocab, dtype, vocab + pad, shift)
    scores = (-np.sort(rng.exponential(2.0, (G, W)).cumsum(1), axis=1)[:, ::-1] - 3).astype(np.float32)
    ids = rng.choice(vocab, min(stops, vocab), replace=False).tolist()
    if ids:
        x[::2, ids[0]] = 9.0
    check_select(ctx, x, scores, n, ids)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two values", "zeros of both signs", "like beams"])
def test_select_ties_and_orders(ctx, dtype, kind):
    """Equal logits go to the lowest token and the lowest beam; rows in rising order raise the bound at every step."""
    import torch

    G, W, n, vocab = 2, 3, 6, 9001
    t = torch.arange(vocab, device="cuda")
    row = {"equal": torch.full((vocab,), 1.5, device="cuda"), "rising": t / 512.0, "falling": -t / 512.0,
           "two values": (t % 7 == 3).float(), "zeros of both signs": torch.where(t % 2 == 0, -0.0, 0.0) - (t % 5 == 1).float(),
           "like beams": torch.sin(t * 1.7) * 6}[kind]
    x = row.to(torch_type(dtype)).repeat(G * W, 1)
    scores = np.array([[-1.0, -1.0, -1.0], [-2.0, -1.0, -1.0]], np.float32)
    log("ties", kind, dtype)
    r = check_select(ctx, x, scores, n, [3, 8999])
    # bit for bit: rows of the same logits have the same sums, so that equal scores are equal
    want = continuations(x.double().cpu().numpy(), scores, W)
    for g in range(G):
        s, a, _, tok = want[g]
        go = [k for k in range(s.size) if tok[k] not in (3, 8999)][:n]
        assert r.token[g].tolist() == tok[go].tolist() and r.parent[g].tolist() == a[go].tolist()


@pytest.mark.parametrize("G,W,n,vocab", [(2, 64, 64, 600), (3, 40, 7, 9000), (1, 64, 64, 70000), (1, 2, 64, 400000)])
def test_select_more_equal_entries_than_are_ranked_at_once(ctx, G, W, n, vocab):
    """Beams and logits that are all alike, but for some: the lists are merged in order."""
    import torch

    x = torch.zeros(G * W, vocab, device="cuda")
    x[:, vocab // 2] = 1.0
    x[-1, 5] = 3.0
    log("alike", G, W, n, vocab)
    r = check_select(ctx, x, np.full((G, W), -2.0, np.float32), n, [0])
    want = continuations(x.double().cpu().numpy(), np.full((G, W), -2.0), W)
    for g in range(G):
        s, a, _, tok = want[g]
        go = np.flatnonzero(tok != 0)[:n]
        assert r.token[g].tolist() == tok[go].tolist() and r.parent[g].tolist() == a[go].tolist()


def test_select_rows_that_are_not_live(ctx):
    """Rows of -inf, with a NaN, with a +inf; scores of -inf, +inf and NaN; groups with fewer continuations than n and
    with none; masked rows that leave one token."""
    import torch

    G, W, n, vocab = 6, 4, 5, 5000
    rng = np.random.default_rng(5)
    x = logits(rng, G * W, vocab, "f32")
    scores = -rng.uniform(1, 5, (G, W)).astype(np.float32)
    scores[0] = [-INF, -3, INF, np.nan]
    x[4:8] = -INF                       # group 1: nothing
    x[8:12] = -INF                      # group 2: a token here and there
    x[8, 77], x[10, 4999], x[10, 0] = 2.0, -1.0, 5.0
    x[12, 100], x[13, 4097], x[14] = float("nan"), INF, float("nan")  # group 3: one live row
    scores[4] = -INF                    # group 4: over
    x[20:24, 1:] = -INF                 # group 5: one token each
    log("not live")
    r = check_select(ctx, x, scores, n, [77, 0])
    assert r.token[1].tolist() == [-1] * n and r.n_end.tolist()[1] == 0
    assert set(r.parent[3].tolist()) == {15} and r.n_end[5] == 4
    for dt in ("bf16", "f16"):
        check_select(ctx, x.to(torch_type(dt)), scores, n, [77, 0])
    # -inf is not a number that a mask leaves: the type's lowest value is one
    low = torch.full((2, 4000), torch.finfo(torch.float32).min, device="cuda")
    low[0, 9] = 1.0
    check_select(ctx, low, np.zeros((1, 2), np.float32), 3)


@pytest.mark.parametrize("stops", [[0, 1, 2], [2, 2, -5, 99, 1 << 30], []])
def test_select_stop_tokens(ctx, stops):
    """Every token a stop; stops named twice or outside the vocabulary; none."""
    import torch

    x = torch.tensor([[1.0, 3.0, 2.0], [0.5, 0.25, 4.0]], device="cuda")
    log("stops", stops)
    r = check_select(ctx, x, np.array([[-1.0, -1.5]], np.float32), 4, stops)
    if stops[:1] == [0]:
        assert r.n_end[0] == 4 and r.token[0].tolist() == [-1] * 4


def test_select_without_ends_and_in_the_c_call(ctx):
    import torch

    x = logits(np.random.default_rng(3), 8, 3001, "f32")
    scores = torch.full((2, 4), -1.0, device="cuda")
    want = ctx.beam_select(x, scores, 4)
    out = torch.full((3, 8), 77, dtype=torch.int32, device="cuda")
    p = out.data_ptr()
    assert V.load_library().vsmp_beam_select(ctx._h, x.data_ptr(), 0, 3001, 2, 4, 3001, scores.data_ptr(), 4, None, 0, p, p + 32,
                                             p + 64, None, None, None, None, None) == 0
    torch.cuda.synchronize()
    for k, name in enumerate(("token", "parent", "score")):
        assert torch.equal(out[k].view(2, 4).view(torch.float32 if k == 2 else torch.int32), getattr(want, name))


def test_select_far_rows(ctx):
    """Rows whose elements lie beyond 2^32 bytes and 2^31 elements."""
    import torch

    ld = (1 << 31) + 12345
    buf = torch.empty(ld + 5000, dtype=torch.float16, device="cuda")
    x = buf.as_strided((2, 5000), (ld, 1))
    x.copy_(logits(np.random.default_rng(8), 2, 5000, "f16"))
    log("far rows")
    check_select(ctx, x, np.array([[-1.0, -1.25]], np.float32), 6, [4])


# ---- rows of states --------------------------------------------------------------------------------------


def parents(rng, groups, width, kind="any"):
    p = rng.integers(0, width, (groups, width))
    if kind == "cycle":
        p = (np.arange(width)[None] + rng.integers(1, max(2, width), (groups, 1))) % width
    if kind == "same":
        p = np.arange(width)[None].repeat(groups, 0)
    return (p + width * np.arange(groups)[:, None]).astype(np.int32).reshape(-1)


def moved(t, parent, width, lens, dim):
    """What reorder_rows leaves of a plane (a numpy array), row by row."""
    out = t.copy()
    for i, p in enumerate(parent):
        if p // width != i // width or p < 0 or p >= len(parent) or p == i:
            continue
        if dim is None:
            out[i] = t[p]
            continue
        n = t.shape[dim] if lens is None else min(max(int(lens[p]), 0), t.shape[dim])
        at = (slice(None),) * (dim - 1) + (slice(0, n),)
        out[i][at] = t[p][at]
    return out


@pytest.mark.parametrize("groups,width,shape,dim,dtype,lens,kind", [
    (1, 1, (3, 5, 8), 2, "bf16", True, "any"),
    (1, 4, (3, 512, 64), 2, "bf16", True, "any"),
    (5, 3, (2, 33, 5), 2, "f32", True, "any"),
    (4, 4, (7, 3), 1, "u8", True, "cycle"),         # tokens of 3 bytes
    (3, 8, (19, 2, 8), 1, "f16", False, "cycle"),
    (2, 16, (2, 40, 24), 2, "bf16", True, "any"),
    (2, 17, (1, 9, 7), 2, "f32", True, "any"),
    (1, 32, (2, 21, 16), 2, "f16", True, "cycle"),
    (2, 33, (3, 11, 5), 2, "u8", True, "any"),
    (1, 64, (1, 50, 12), 2, "f32", True, "cycle"),
    (3, 5, (1000,), None, "f32", False, "any"),      # whole rows
    (2, 6, (), None, "i32", False, "cycle"),         # one number a row
    (40000, 2, (3,), None, "i32", False, "any"),     # more groups than a launch counts
    (3, 4, (2, 16, 8), 2, "f32", True, "same"),
])
def test_reorder(ctx, groups, width, shape, dim, dtype, lens, kind):
    import torch

    log("reorder", groups, width, shape, dtype)
    rng = np.random.default_rng(groups + width)
    R = groups * width
    planes = [torch.randint(0, 200, (R,) + shape, device="cuda").to(torch_type(dtype)) for _ in range(3)]
    p = parents(rng, groups, width, kind)
    if R > 4:
        p[1], p[2] = -3, R + 7  # outside: the row stays
        p[3] = (p[3] + width) % R
    n = rng.integers(0, shape[dim - 1] + 1, R).astype(np.int32) if lens else None
    if lens and R > 2:
        n[0], n[-1] = -4, 1 << 30  # taken for nothing and for all
    was = [t.float().cpu().numpy() for t in planes]
    ctx.reorder_rows(V.Planes(planes, token_dim=dim), i32(p), width, lens=i32(n) if lens else None)
    for t, w in zip(planes, was):
        np.testing.assert_array_equal(t.float().cpu().numpy(), moved(w, p, width, n, dim))


@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_reorder_strides_and_addresses(ctx, shift):
    """Planes that start anywhere, rows with room between them, rows within pieces ([heads, rows, tokens, width]); what lies
    between is left as it is."""
    import torch

    rng = np.random.default_rng(shift)
    W, G, H, Tk, D = 4, 3, 3, 10, 6
    R = W * G
    p = parents(rng, G, W)
    n = rng.integers(0, Tk + 1, R).astype(np.int32)
    log("reorder strides", shift)
    for layout in ("rows", "pieces"):
        bufs = [torch.randint(0, 255, (20000,), dtype=torch.uint8, device="cuda") for _ in range(2)]
        strides = (H * (Tk * D + 7) + 5, Tk * D + 7, D, 1) if layout == "rows" else (Tk * D + 3, R * (Tk * D + 3) + 11, D, 1)
        views = [b[shift:].as_strided((R, H, Tk, D), strides, storage_offset=b.storage_offset() + shift) for b in bufs]
        was = [b.cpu().numpy().copy() for b in bufs]
        rows = [v.cpu().numpy().copy() for v in views]
        ctx.reorder_rows(V.Planes(views, token_dim=2), i32(p), W, lens=i32(n))
        for b, v, w, r in zip(bufs, views, was, rows):
            np.testing.assert_array_equal(v.cpu().numpy(), moved(r, p, W, n, 2))
            host = torch.from_numpy(w)
            host[shift:].as_strided((R, H, Tk, D), strides, storage_offset=shift).copy_(torch.from_numpy(moved(r, p, W, n, 2)))
            np.testing.assert_array_equal(b.cpu().numpy(), host.numpy())


def test_reorder_far_rows(ctx):
    """Rows 3 GB apart, pieces of 40 MB."""
    import torch

    far = 3 << 30
    buf = torch.empty(3 * far + (40 << 20), dtype=torch.uint8, device="cuda")
    x = buf.as_strided((4, 40 << 20), (far, 1))
    for i in range(4):
        x[i].fill_(i + 1)
    log("reorder far")
    ctx.reorder_rows(V.Planes([x]), i32([2, 0, 2, 1]), 4)
    assert [int(x[i].min()) for i in range(4)] == [3, 1, 3, 2] == [int(x[i].max()) for i in range(4)]


def test_reorder_more_than_the_caches_hold(ctx):
    """700 MB, whose stores are streamed."""
    import torch

    n = 175 << 20
    x = torch.empty(4, n, dtype=torch.uint8, device="cuda")
    for i in range(4):
        x[i].random_(50 * i, 50 * i + 50, generator=torch.Generator(device="cuda").manual_seed(i))
    sums = [int(x[i].to(torch.int64).sum()) for i in range(4)]
    log("reorder 700 MB")
    ctx.reorder_rows(V.Planes([x]), i32([3, 0, 0, 2]), 4)
    assert [int(x[i].to(torch.int64).sum()) for i in range(4)] == [sums[k] for k in (3, 0, 0, 2)] and torch.equal(x[1], x[2])


# ---- a cache in pages ------------------------------------------------------------------------------------


class Model:
    """A cache in pages row by row: its state, and what every row's tokens are."""

    def __init__(self, rows, row_pages, n_pages, T):
        self.T, self.P, self.cap = T, n_pages, row_pages
        self.table = [[] for _ in range(rows)]
        self.tokens = [[] for _ in range(rows)]
        self.ref = [0] * n_pages

    def step(self, parent, add):
        T, ref = self.T, list(self.ref)
        rows = []
        for t in self.table:
            for q in t:
                ref[q] -= 1
        for i, p in enumerate(parent):
            there = 0 <= p < len(self.table)
            toks, pages = (list(self.tokens[p]), list(self.table[p])) if there else ([], [])
            want = max(0, len(toks) + int(add[i]))
            ok = want <= self.cap * T
            if ok and want < len(toks):
                toks, pages = toks[:want], pages[:-(-want // T)]
            rows.append([toks, pages, want if ok else len(toks), ok])
            for q in pages:
                ref[q] += 1
        grow = {}
        for i, (toks, pages, want, ok) in enumerate(rows):
            if want > len(toks) and len(toks) % T:
                grow.setdefault(pages[-1], []).append(i)
        keep = {q: sorted(w, key=lambda i: (-len(rows[i][0]), i))[0] for q, w in grow.items() if ref[q] == len(w)}
        free = [q for q in range(self.P) if ref[q] <= 0]
        asked, copies = 0, []
        for i, r in enumerate(rows):
            toks, pages, want, ok = r
            if want <= len(toks):
                continue
            away = len(toks) % T > 0 and keep.get(pages[-1]) != i
            need = -(-want // T) - len(pages) + away
            asked += need
            if need and asked > len(free):
                r[2], r[3] = len(toks), False
                continue
            got = free[asked - need:asked]
            if away:
                copies.append((pages[-1], got[0], len(toks) % T))
                ref[pages.pop()] -= 1
            for q in got:
                ref[q] = 1
            pages += got
        self.table, self.ref = [r[1] for r in rows], ref
        self.tokens, grown = [r[0] for r in rows], [r[2] - len(r[0]) for r in rows]
        return [int(r[3]) for r in rows], grown, copies

    def compact(self):
        live = [q for q in range(self.P) if self.ref[q] > 0]
        n = len(live)
        to = {q: q for q in live}
        to.update(zip([q for q in live if q >= n], [q for q in range(n) if self.ref[q] <= 0]))
        ref = [0] * self.P
        for q in live:
            ref[to[q]] = self.ref[q]
        self.ref, self.table = ref, [[to[q] for q in t] for t in self.table]
        return [to.get(q, -1) for q in range(self.P)], n


class Cache:
    """A model and the framework's cache beside it; every plane holds the tokens' numbers."""

    def __init__(self, ctx, rows, row_pages, n_pages, T, heads=2, width=3, planes=2, by_head=False, dtype="i32"):
        import torch

        self.ctx, self.m, self.by_head = ctx, Model(rows, row_pages, n_pages, T), by_head
        shape = (n_pages, heads, T, width) if by_head else (n_pages, T, heads, width)
        self.planes = [torch.full(shape, 255 if dtype == "u8" else -9, dtype=torch_type(dtype), device="cuda") for _ in range(planes)]
        self.cache = V.Planes(self.planes, token_dim=2 if by_head else 1)
        self.pages = V.Pages.empty(rows, row_pages, n_pages, T)
        self.next, self.mod = 0, 250 if dtype == "u8" else 1 << 30

    def check(self):
        p, m = self.pages, self.m
        table, lens, ref = p.table.cpu().numpy(), p.lens.cpu().numpy(), p.ref.cpu().numpy()
        assert lens.tolist() == [len(t) for t in m.tokens]
        for i, t in enumerate(m.table):
            assert table[i].tolist() == t + [-1] * (table.shape[1] - len(t)), i
        assert ref.tolist() == m.ref
        host = [x.cpu().numpy() for x in self.planes]
        if self.by_head:
            host = [x.swapaxes(1, 2) for x in host]
        for k, x in enumerate(host):
            for i, toks in enumerate(m.tokens):
                if toks:
                    got = x[m.table[i]].reshape((-1,) + x.shape[2:])[:len(toks)]
                    assert (got == np.array(toks)[:, None, None]).all(), (k, i)

    def write(self, grown):
        """The grown rows' new tokens, as a model's attention writes them: only behind what the row had."""
        import torch

        for i, n in enumerate(grown):
            for _ in range(max(n, 0)):
                at, tok = len(self.m.tokens[i]), self.next % self.mod
                self.next += 1
                q, t = self.m.table[i][at // self.m.T], at % self.m.T
                for x in self.planes:
                    (x[q, :, t] if self.by_head else x[q, t]).fill_(tok)
                self.m.tokens[i].append(tok)
        torch.cuda.synchronize()

    def step(self, parent, add, **kw):
        want = self.m.step(range(len(self.m.table)) if parent is None else parent, [add] * len(self.m.table) if isinstance(add, int) else add)
        self.pages, ok = self.ctx.pages_step(self.pages, None if parent is None else i32(parent), add if isinstance(add, int) else i32(add),
                                             cache=self.cache, **kw)
        assert ok.cpu().numpy().tolist() == want[0]
        lens = self.pages.lens.cpu().numpy()
        for i, toks in enumerate(self.m.tokens):
            assert lens[i] == len(toks) + max(want[1][i], 0)
        self.write(want[1])
        self.check()
        return want

    def compact(self):
        moved, n = self.m.compact()
        self.pages, got, live = self.ctx.pages_compact(self.pages, cache=self.cache)
        assert got.cpu().numpy().tolist() == moved and live.item() == n
        self.check()


@pytest.mark.parametrize("rows,row_pages,n_pages,T,by_head,dtype", [
    (4, 6, 16, 4, False, "i32"),     # short of pages again and again
    (6, 8, 60, 3, True, "i32"),
    (5, 40, 200, 1, False, "u8"),    # pages of one token: none is ever begun
    (8, 5, 64, 16, True, "f32"),
    (1, 3, 2, 5, False, "i32"),
    (33, 4, 4500, 8, False, "i32"),  # more pages than one workgroup's
    (12, 9, 65536, 2, False, "i32"),
    (9, 9, 65537, 2, False, "i32"),  # a pool whose step is more than one launch
    (1025, 3, 1500, 2, False, "i32"),
])
def test_pages_any_steps(ctx, rows, row_pages, n_pages, T, by_head, dtype):
    """Thirty steps of any kind: forks, cuts, ends, growth by one token and by several pages, rows that do not fit."""
    log("pages", rows, n_pages, T)
    rng = np.random.default_rng(rows * 100 + T)
    c = Cache(ctx, rows, row_pages, n_pages, T, by_head=by_head, dtype=dtype)
    for k in range(30 if rows < 100 else 4):
        parent = rng.integers(-1, rows + (k % 5 == 4), rows) if k % 3 else rng.integers(0, rows, rows)
        add = rng.choice([-T - 1, -1, 0, 1, 1, 1, 2, T, 3 * T + 1], rows)
        if k % 7 == 6:
            parent, add = None, int(rng.integers(-2, 3))
        c.step(parent, add)
        if k % 10 == 9:
            c.compact()


def test_pages_search(ctx):
    """Beams of searches over many steps: every row grows by one token from a parent of its group."""
    rng = np.random.default_rng(2)
    G, W = 5, 4
    c = Cache(ctx, G * W, 16, 300, 4)
    c.step([-1] * (G * W), [int(rng.integers(1, 20)) if i % W == 0 else 0 for i in range(G * W)])
    c.step([i - i % W for i in range(G * W)], 1)
    copies = 0
    for k in range(20):
        copies += len(c.step(parents(rng, G, W), 1)[2])
    log("copies", copies)
    assert copies > 20
    c.compact()
    c.step([-1] * (G * W), 0)
    assert sum(c.m.ref) == 0


def test_pages_rows_of_other_numbers(ctx):
    """A state of three rows becomes one of eight, and one of two: rows that are dropped give up their pages."""
    c = Cache(ctx, 3, 8, 40, 4)
    c.step([-1, -1, -1], [9, 0, 16])
    c.step([0, 0, 0, 1, 2, 2, 2, -1], [1, 1, 0, 3, 1, -5, 1, 6])
    c.step([5, 0], 1)
    c.step(None, 1)


def test_pages_holders_outside_the_tables(ctx):
    """A caller's own hold on a page: a row that grows in it copies it, and it is not given out while held."""
    c = Cache(ctx, 2, 4, 6, 4)
    c.step([-1, -1], [6, 0])
    q = c.m.table[0][1]
    c.m.ref[q] += 1
    c.pages.ref[q] += 1
    assert len(c.step(None, [1, 0])[2]) == 1
    c.step([-1, -1], [0, 0])
    assert c.m.ref[q] == 1
    c.step(None, [16, 4])   # all that are free: the held one is not among them
    assert c.m.ref[q] == 1 and q not in c.m.table[0] + c.m.table[1]


def test_pages_writers_of_one_page(ctx):
    """A begun page of a longer row and a shorter one (a cut fork): the longer keeps it when both grow; neither does where
    a third holds on to it."""
    c = Cache(ctx, 3, 4, 12, 8)
    c.step([-1, -1, -1], [7, 0, 0])
    c.step([0, 0, -1], [0, -2, 0])
    want = c.step([1, 0, -1], [1, 1, 0])      # row 0 has 5 tokens, row 1 has 7: row 0 copies
    assert [x[2] for x in want[2]] == [5]
    c.step([1, 1, 1], [0, 0, 0])
    c = Cache(ctx, 3, 4, 12, 8)
    c.step([-1, -1, -1], [5, 0, 0])
    assert len(c.step([0, 0, 0], [1, 1, 0])[2]) == 2


def test_pages_no_page_left_keeps_a_shared_one_whole(ctx):
    """Two rows share a begun page and one page is short: the row that gets none keeps its tokens whatever the other
    writes."""
    c = Cache(ctx, 3, 4, 2, 4)
    c.step([-1, -1, -1], [3, 4, 0])
    assert c.m.ref == [1, 1]
    want = c.step([0, 1, 0], [1, 0, 1])       # rows 0 and 2 share page 0; no free page
    assert want[0] == [1, 1, 0]
    c.step([2, -1, 0], [0, 0, 0])


def test_pages_far_and_large(ctx):
    """The largest pool and the most rows: 2^20 pages, 8,192 rows of which most grow."""
    import torch

    P, R, T = 1 << 20, 8192, 4
    log("largest pool")
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 40, R)
    n = -(-lens // T)
    ids = rng.permutation(P)[:n.sum()]
    table = np.full((R, 12), -1, np.int32)
    table[np.arange(12)[None] < n[:, None]] = ids
    ref = np.zeros(P, np.int32)
    ref[ids] = 1
    rest = np.flatnonzero(ref == 0)
    held = rest[rng.random(rest.size) < 0.97]
    ref[held] = 1                              # the caller's: the free ones lie apart
    planes = [torch.arange(P * T, dtype=torch.int32, device="cuda").view(P, T, 1)]
    m = Model(R, 12, P, T)
    m.table = [table[i, :n[i]].tolist() for i in range(R)]
    m.tokens = [[0] * int(k) for k in lens]
    m.ref = ref.tolist()
    parent = np.where(rng.random(R) < 0.5, np.arange(R), rng.integers(-1, R, R))
    add = rng.integers(-2, 4, R)
    ok, grown, copies = m.step(parent, add)
    pages = V.Pages(i32(table), i32(lens), i32(ref), T)
    to, got = ctx.pages_step(pages, i32(parent), i32(add), cache=V.Planes(planes, token_dim=1))
    assert got.cpu().numpy().tolist() == ok and to.ref.cpu().numpy().tolist() == m.ref
    assert to.lens.cpu().numpy().tolist() == [len(t) + g for t, g in zip(m.tokens, grown)]
    want = np.full((R, 12), -1)
    for i, t in enumerate(m.table):
        want[i, :len(t)] = t
    np.testing.assert_array_equal(to.table.cpu().numpy(), want)
    x = planes[0].cpu().numpy().reshape(P, T)
    for src, dst, k in copies:
        assert (x[dst, :k] == src * T + np.arange(k)).all() and (x[dst, k:] == dst * T + np.arange(k, T)).all()
    moved, live = m.compact()
    planes[0].copy_(torch.arange(P * T, dtype=torch.int32, device="cuda").view(P, T, 1))
    to2, mv, nl = ctx.pages_compact(to, cache=V.Planes(planes, token_dim=1))
    assert nl.item() == live and to2.ref.cpu().numpy().tolist() == m.ref
    moved = np.array(moved)
    np.testing.assert_array_equal(mv.cpu().numpy(), moved)
    x = planes[0].cpu().numpy().reshape(P, T)
    src = np.flatnonzero(moved >= 0)
    np.testing.assert_array_equal(x[moved[src]], src[:, None] * T + np.arange(T))


@pytest.mark.parametrize("rows,row_pages", [(8192, 1 << 20), (3000, 40)])
def test_pages_rows_that_ask_for_more_than_there_is(ctx, rows, row_pages):
    """Rows that want up to 2^30 tokens each, together more than 32 bits count: the first ones that fit get their pages,
    none of the others any."""
    import torch

    P = 1000
    table = torch.full((1, row_pages), -1, dtype=torch.int32, device="cuda")
    pages = V.Pages(table.expand(1, row_pages), i32([0]), i32(np.zeros(P)), 1 if row_pages > 40 else 1 << 24)
    T = pages.page_tokens
    n = 64 if row_pages > 40 else rows  # (8,192 rows of 2^20 entries would take 32 GB)
    to = V.Pages(torch.empty(n, row_pages, dtype=torch.int32, device="cuda"), i32(np.zeros(n)), i32(np.zeros(P)), T)
    want = np.full(n, row_pages * T if row_pages > 40 else 40 * T)
    want[:2] = 5 * T, 7 * T
    log("more than there is", rows, row_pages)
    got, ok = ctx.pages_step(pages, i32(np.full(n, -1)), i32(want), out=to)
    need = -(-want // T)
    fits = np.cumsum(need) <= P
    assert ok.cpu().numpy().tolist() == fits.astype(int).tolist()
    assert got.lens.cpu().numpy().tolist() == np.where(fits, want, 0).tolist()
    assert int(got.ref.sum()) == int(need[fits].sum())


def test_pages_tables_with_numbers_that_are_no_pages(ctx):
    """Entries outside the pool stand for no page: nothing is read or counted through them, and rows go on with them."""
    P, T = 10, 4
    table = np.array([[3, -7, 1 << 30], [P, 2, -1]], np.int32)
    ref = np.zeros(P, np.int32)
    ref[[3, 2]] = 1
    import torch

    x = torch.arange(P * T, dtype=torch.int32, device="cuda").view(P, T, 1)
    pages = V.Pages(i32(table), i32([10, 99]), i32(ref), T)   # 99: taken for the row's room, 12 tokens
    log("bad pages")
    to, ok = ctx.pages_step(pages, i32([1, 0]), i32([0, 1]), cache=V.Planes([x], token_dim=1))
    assert to.table.cpu().numpy().tolist() == [[P, 2, -1], [3, -7, 1 << 30]] and to.lens.tolist() == [12, 11]
    assert to.ref.tolist() == ref.tolist() and ok.tolist() == [1, 1]
    to, moved, live = ctx.pages_compact(pages, cache=V.Planes([x], token_dim=1))
    assert to.table.cpu().numpy().tolist() == [[1, -7, 1 << 30], [P, 0, -1]] and to.lens.tolist() == [10, 12]
    assert live.item() == 2 and moved.tolist() == [-1, -1, 0, 1] + [-1] * 6


@pytest.mark.parametrize("n_pages", [1, 63, 64, 65, 4096, 4097])
def test_compact_pools(ctx, n_pages):
    """Pools whose last word is not whole; nothing live, everything live, one page."""
    import torch

    rng = np.random.default_rng(n_pages)
    for share in (0.0, 0.3, 0.9, 1.0):
        ref = (rng.random(n_pages) < share).astype(np.int32) * rng.integers(1, 4, n_pages)
        ref[rng.random(n_pages) < 0.05] -= 4  # below 0: free
        x = torch.arange(n_pages * 2, dtype=torch.int32, device="cuda").view(n_pages, 2)
        m = Model(1, 1, n_pages, 2)
        m.ref = ref.tolist()
        log("compact", n_pages, share)
        moved, n = m.compact()
        pages = V.Pages(i32([[-1]]), i32([0]), i32(ref), 2)
        to, got, live = ctx.pages_compact(pages, cache=V.Planes([x], token_dim=1))
        moved = np.array(moved)
        assert live.item() == n and to.ref.cpu().numpy().tolist() == m.ref
        np.testing.assert_array_equal(got.cpu().numpy(), moved)
        src = np.flatnonzero(moved >= 0)
        np.testing.assert_array_equal(x.cpu().numpy()[moved[src]], src[:, None] * 2 + np.arange(2))


# ---- together --------------------------------------------------------------------------------------------


def test_a_step_in_a_graph_beside_eager_work(ctx):
    """Selection, rows and pages of a step captured once and replayed on new inputs, with eager calls of the same
    context between the replays, against the same step made eagerly."""
    import torch

    G, W, vocab, T = 3, 4, 20011, 4
    R = G * W
    rng = np.random.default_rng(4)
    x = logits(rng, R, vocab, "f32")
    scores = torch.full((G, W), -1.0, device="cuda")
    state = torch.randn(R, 2, 9, 5, device="cuda")
    planes = V.Planes([state], token_dim=2)
    pool = torch.randn(200, T, 6, device="cuda")
    cache = V.Planes([pool], token_dim=1)
    start = V.Pages.empty(R, 8, 200, T)
    start, _ = ctx.pages_step(start, add=6)
    to = start.like()
    keep = {}

    def step():
        keep["sel"] = ctx.beam_select(x, scores, W, stop_ids=[7])
        ctx.reorder_rows(planes, keep["sel"].parent.view(-1), W)
        keep["to"], keep["ok"] = ctx.pages_step(start, keep["sel"].parent.view(-1), 1, cache=cache, out=to)
        keep["compact"] = ctx.pages_compact(to, cache=cache)

    def seen():
        torch.cuda.synchronize()
        c = keep["compact"]
        return [t.clone() for t in (*keep["sel"], state, to.table, to.lens, to.ref, keep["ok"], c[0].table, c[0].ref, c[1], c[2], pool)]

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    captured = dict(keep)
    for k in range(4):
        fresh = logits(np.random.default_rng(50 + k), R, vocab, "f32")
        s0, p0 = torch.randn_like(state), torch.randn_like(pool)
        x.copy_(fresh)
        state.copy_(s0)
        pool.copy_(p0)
        log("replay", k)
        g.replay()
        keep = dict(captured)
        got = seen()
        state.copy_(s0)
        pool.copy_(p0)
        step()
        for a, b in zip(got, seen()):
            assert torch.equal(a, b)
        scores.copy_(-torch.rand(G, W, device="cuda").sort(1).values * 3)


def test_a_first_call_in_a_capture_is_refused():
    """A context without the operators' scratch would have to allocate it: refused with a message, and the capture goes on."""
    import torch

    fresh = V.Context(0)
    x, scores = torch.zeros(2, 100, device="cuda"), torch.zeros(1, 2, device="cuda")
    pages, to = V.Pages.empty(2, 4, 10, 4), V.Pages.empty(2, 4, 10, 4)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = x + 1
        for call in (lambda: fresh.beam_select(x, scores), lambda: fresh.pages_step(pages, add=1, out=to),
                     lambda: fresh.pages_compact(pages, out=to)):
            with pytest.raises(V.VsmpError, match="before capturing"):
                call()
    g.replay()
    torch.cuda.synchronize()
    assert y[0, 0].item() == 1.0


def test_python_refuses_what_is_not_a_cache(ctx):
    """Planes and pages of other shapes, strides, types and sizes than the operators take."""
    import torch

    x = torch.zeros(4, 3, 8, 5, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    for make, words in (
        (lambda: V.Planes([x, x]), "of their own"),
        (lambda: V.Planes([x, torch.zeros(4, 3, 8, 4, device="cuda")]), "one shape"),
        (lambda: V.Planes([x, x.clone().half()]), "one shape"),
        (lambda: V.Planes([x], token_dim=4), "token_dim"),
        (lambda: V.Planes([x], token_dim=0), "token_dim"),
        (lambda: V.Planes([x.transpose(2, 3)], token_dim=2), "side by side"),
        (lambda: V.Planes([x[:, :, :, ::2]], token_dim=2), "side by side"),
        (lambda: V.Planes([torch.zeros(4, 3, 2, 16, 5, device="cuda")[:, :, :, ::2]], token_dim=3), "side by side"),
        (lambda: V.Planes([torch.zeros(4, 3, 4, 8, 5, device="cuda")[:, :, :3]], token_dim=3), "one stride"),
        (lambda: V.Planes([x[:0]]), "at least one"),
        (lambda: V.Pages(i, i, i, 4), "2-D int32"),
        (lambda: V.Pages(torch.zeros(4, 2, device="cuda"), i, i, 4), "2-D int32"),
        (lambda: V.Pages(torch.zeros(2, 4, dtype=torch.int32, device="cuda").t(), i, i, 4), "contiguous rows"),
        (lambda: V.Pages(torch.zeros(3, 4, dtype=torch.int32, device="cuda"), i, i, 4), "an entry for each row"),
        (lambda: V.Pages(torch.zeros(4, 4, dtype=torch.int32, device="cuda"), i.float(), i, 4), "lens"),
        (lambda: V.Pages(torch.zeros(4, 4, dtype=torch.int32, device="cuda"), i.view(2, 2), i, 4), "one-dimensional"),
        (lambda: ctx.beam_select(torch.zeros(4, 10, device="cuda"), torch.zeros(4, device="cuda")), "scores"),
        (lambda: ctx.beam_select(torch.zeros(4, 10, device="cuda"), torch.zeros(1, 3, device="cuda")), "scores"),
        (lambda: ctx.beam_select(torch.zeros(4, 10, device="cuda"), torch.zeros(1, 4, device="cuda").double()), "scores"),
        (lambda: ctx.beam_select(torch.zeros(4, 10, device="cuda").double(), torch.zeros(1, 4, device="cuda")), "float32, bfloat16"),
        (lambda: ctx.beam_select(torch.zeros(4, 10, device="cuda"), torch.zeros(1, 4, device="cuda"), 0), "n >= 1"),
        (lambda: ctx.beam_select(torch.zeros(4, 10, device="cuda"), torch.zeros(1, 4, device="cuda"), 4, range(17)), "n_stop"),
        (lambda: ctx.reorder_rows(V.Planes([x]), i.long(), 4), "parent"),
        (lambda: ctx.reorder_rows(V.Planes([x]), i[:3], 4), "parent"),
        (lambda: ctx.reorder_rows(V.Planes([x]), i, 3), "width"),
        (lambda: ctx.pages_step(V.Pages.empty(4, 2, 4, 4), add=i.float()), "add"),
        (lambda: ctx.pages_step(V.Pages.empty(4, 2, 4, 4), cache=V.Planes([x], token_dim=2)), "page_tokens tokens"),
    ):
        with pytest.raises(V.VsmpError, match=words):
            make()
    p = V.Pages.empty(4, 2, 4, 4)
    with pytest.raises(V.VsmpError, match="must not overlap"):
        ctx.pages_step(p, add=1, out=p)


def test_on_another_stream(ctx):
    """Inputs made on a stream that is busy, the calls on it, outputs that are its memory."""
    import torch

    st = torch.cuda.Stream()
    rng = np.random.default_rng(9)
    x = logits(rng, 8, 30011, "bf16")
    scores = np.full((2, 4), -1.0, np.float32)
    want = check_select(ctx, x, scores, 4, [5])
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            a = a @ a * 1e-3
        y = (x.float() + 0 * a[:1, :1].nan_to_num(0, 0, 0)).to(torch.bfloat16)
        s = torch.from_numpy(scores).cuda()
    got = ctx.beam_select(y, s, 4, stop_ids=[5], stream=st)
    pages = V.Pages.empty(4, 4, 30, 4)
    torch.cuda.synchronize()
    to, ok = ctx.pages_step(pages, add=5, stream=st)
    to2, moved, live = ctx.pages_compact(to, stream=st)
    st.synchronize()
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.cpu().numpy(), b)
    assert ok.tolist() == [1] * 4 and to2.lens.tolist() == [5] * 4 and live.item() == 8
