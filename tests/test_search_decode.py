"""BeamDecoder: searches over a model whose logits depend on every id before them, read back from the cache in pages or from
the states held row by row that the search moved, against a search in 64 bits over plain lists."""
import numpy as np
import pytest

import verbo_amd as V
from verbo_amd import decode


def model(vocab, seed, sharp=2.0):
    """Logits of the next id from all ids so far: a fixed pseudo-random row for each sequence."""
    def logits(ids):
        h = seed
        for t in ids:
            h = (h * 1000003 + int(t) + 7) & 0x7FFFFFFF
        return np.random.RandomState(h).normal(0, sharp, vocab).astype(np.float32)
    return logits


def plain_search(logits, prompt, width, max_tokens, stops, penalty):
    """The search by its definition: beams as lists of ids, scores in 64 bits from scores kept in fp32."""
    beams, ended = [(np.float32(0.0), [])], []
    for t in range(max_tokens):
        found = []
        for b, (score, ids) in enumerate(beams):
            x = logits(list(prompt) + ids).astype(np.float64)
            top = x.max()
            lse = top + np.log(np.exp(x - top).sum())
            found += [(-(float(score) + (x[k] - lse)), b, -x[k], k) for k in range(x.size) if x[k] > -np.inf]
        found.sort()
        length = float(t + 1) ** penalty
        for s, b, _, k in found[:width]:
            if k in stops:
                ended.append((float(np.float32(-s)) / length, beams[b][1]))
        ended = sorted(ended, key=lambda e: -e[0])[:width]
        beams = [(np.float32(-s), beams[b][1] + [k]) for s, b, _, k in found if k not in stops][:width]
        if not beams or (len(ended) == width and ended[-1][0] >= float(beams[0][0]) / length):
            return ended
        if t + 1 == max_tokens:
            ended = sorted(ended + [(float(s) / length, ids) for s, ids in beams], key=lambda e: -e[0])[:width]
    return ended


def test_decoder_refuses():
    for width, vocab in ((0, 10), (65, 10), (4, 0)):
        with pytest.raises(V.VsmpError):
            decode.BeamDecoder(width, vocab)


def test_the_plain_search_finds_the_best_of_a_small_tree():
    """With a beam for every prefix the search is exhaustive."""
    logits = model(3, 5)
    best = plain_search(logits, [1], 9, 2, (), 1.0)
    every = []
    for a in range(3):
        for b in range(3):
            s = 0.0
            for ids, k in (([], a), ([a], b)):
                x = logits([1] + ids).astype(np.float64)
                s += x[k] - np.log(np.exp(x).sum())
            every.append((s / 2, [a, b]))
    every.sort(key=lambda e: -e[0])
    assert [e[1] for e in best] == [e[1] for e in every]


class Recall:
    """A model that reads its past from the states that the search moved. pages: a plane of ids in pages; rows: a
    plane of ids [rows, tokens, 1]; and that keeps, of its own, only the logits' rule."""

    def __init__(self, logits, prompts, width, room, paged, page=4):
        import torch

        self.logits, self.prompts, self.width, self.paged = logits, prompts, width, paged
        G, n = len(prompts), max(len(p) for p in prompts)
        if paged:
            cap = -(-(n + room) // page) + 1
            self.pool = torch.full((G * (width + 1) * cap, page, 1), -5, dtype=torch.int32, device="cuda")
            self.cache = V.Planes([self.pool], token_dim=1)
            ctx = V.Context(0)
            empty = V.Pages.empty(G, cap, self.pool.shape[0], page)
            self.start, ok = ctx.pages_step(empty, add=torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda"))
            assert bool(ok.all())
            for g, p in enumerate(prompts):
                for k, t in enumerate(p):
                    self.pool[self.start.table[g, k // page], k % page, 0] = int(t)
            torch.cuda.synchronize()
        else:
            self.ids = torch.full((G * width, n + room, 1), -5, dtype=torch.int32, device="cuda")
            self.states = V.Planes([self.ids], token_dim=1)
            for g, p in enumerate(prompts):
                self.ids[g * width, :len(p), 0] = torch.tensor(p, dtype=torch.int32)
        self.page = page

    def __call__(self, step, tokens, pages):
        import torch

        rows = []
        if step == 0:
            rows = [list(p) for p in self.prompts]
        else:
            last = tokens.cpu().numpy()
            if self.paged:
                table, lens = pages.table.cpu().numpy(), pages.lens.cpu().numpy()
                for i, t in enumerate(last):
                    if t >= 0:
                        at = int(lens[i]) - 1
                        self.pool[int(table[i, at // self.page]), at % self.page, 0] = int(t)
                pool = self.pool.cpu().numpy()
                for i, t in enumerate(last):
                    n = int(lens[i])
                    assert (n > 0) == (t >= 0)
                    rows.append(pool[table[i, :-(-n // self.page)]].reshape(-1)[:n].tolist() if t >= 0 else None)
            else:
                for i, t in enumerate(last):
                    n = len(self.prompts[i // self.width]) + step
                    if t >= 0:
                        self.ids[i, n - 1, 0] = int(t)
                    rows.append(self.ids[i, :n, 0].cpu().numpy().tolist() if t >= 0 else None)
        nothing = np.full(self.vocab, np.nan, np.float32)  # of a beam that is not live nothing is read
        return torch.from_numpy(np.stack([self.logits(r) if r is not None else nothing for r in rows])).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("width,vocab,max_tokens,stops,penalty", [
    (1, 40, 9, (3,), 1.0),
    (4, 50, 12, (3, 7), 1.0),
    (5, 7, 10, (2,), 0.0),
    (3, 200, 8, (), 2.0),
    (8, 5, 6, (0, 1, 2, 3), 1.0),   # most continuations end
    (3, 2, 5, (0, 1), 1.0),         # all do
])
@pytest.mark.parametrize("paged", [True, False])
def test_search(width, vocab, max_tokens, stops, penalty, paged):
    from helpers import log

    rng = np.random.default_rng(width * 100 + vocab)
    prompts = [rng.integers(0, vocab, int(rng.integers(1, 11))).tolist() for _ in range(3)]
    logits = model(vocab, width + vocab)
    m = Recall(logits, prompts, width, max_tokens, paged)
    m.vocab = vocab
    log("search", width, vocab, paged)
    dec = decode.BeamDecoder(width, vocab)
    got = dec.search(prompts, m, max_tokens, stops, penalty, **(dict(pages=m.start, cache=m.cache) if paged else dict(states=m.states)))
    for p, res in zip(prompts, got):
        want = plain_search(logits, p, width, max_tokens, stops, penalty)
        assert [ids for ids, _ in res] == [ids for _, ids in want]
        # a step's score is off by its row's sum (2e-7 of exponentials at most 40 below the largest, added in fp32 over
        # fewer than 256 logits: 340 * 2^-24) and by its rounding
        np.testing.assert_allclose([s for _, s in res], [s for s, _ in want], rtol=0, atol=max_tokens * (340 + 64) * 2.0 ** -24)
    if paged:
        assert int(dec.pages.ref.abs().sum()) == 0 and int(dec.pages.lens.sum()) == 0


@pytest.mark.gpu
def test_search_says_when_the_pool_is_short():
    m = Recall(model(30, 1), [[1, 2, 3]], 4, 20, True)
    m.vocab = 30
    full = V.Pages(m.start.table, m.start.lens, m.start.ref.clone().fill_(1), 4)
    with pytest.raises(V.VsmpError, match="no page left"):
        decode.BeamDecoder(4, 30).search([[1, 2, 3]], m, 20, pages=full, cache=m.cache)


@pytest.mark.gpu
def test_search_of_width_one_is_greedy():
    """The ids that the framework's own greedy decoding picks."""
    import torch

    logits = model(64, 9)
    prompts = [[1, 2], [5]]
    rows = {}

    def own(step, tokens, pages):
        if step == 0:
            rows.clear()
            rows.update({g: list(p) for g, p in enumerate(prompts)})
        else:
            for g, t in enumerate(tokens.tolist()):
                rows[g].append(t)
        return torch.from_numpy(np.stack([logits(rows[g]) for g in range(2)])).cuda()

    def batch(step, last, live):
        return own(step, torch.from_numpy(last) if step else None, None)

    got = decode.BeamDecoder(1, 64).search(prompts, own, 7)
    want = decode.BatchDecoder([decode.Opts(max_tokens=7, temp=0.0)] * 2, 64).generate(prompts, batch)
    assert [r[0][0] for r in got] == [t for t, _ in want]


def holders(pages):
    """How many rows hold each page, from the tables."""
    table, lens = pages.table.cpu().numpy(), pages.lens.cpu().numpy()
    out = np.zeros(pages.ref.numel(), int)
    for row, n in zip(table, lens):
        np.add.at(out, row[:-(-int(n) // pages.page_tokens)], 1)
    return out


@pytest.mark.gpu
def test_the_state_of_a_search_that_raised_owns_its_pages():
    """One search ends at once and its pages go to the other's beams, then the pool is short: what self.pages holds is
    the state whose rows own the pages, and giving those rows up empties the pool."""
    import torch

    prompts = [[1, 2, 3], [4, 5, 6]]

    def logits(ids):
        x = model(30, 2)(ids)
        if len(ids) == 3 and ids[0] == 1:
            x[[7, 8]] = 50.0  # both beams of the first prompt end here
        return x

    m = Recall(logits, prompts, 2, 6, True, page=1)
    m.vocab = 30
    P = 10  # three tokens of each prompt, and four more
    ctx = V.Context(0)
    m.pool = torch.full((P, 1, 1), -5, dtype=torch.int32, device="cuda")
    m.cache = V.Planes([m.pool], token_dim=1)
    m.start, ok = ctx.pages_step(V.Pages.empty(2, 10, P, 1), add=3)
    assert bool(ok.all()) and m.start.table[0, :3].tolist() == [0, 1, 2]
    m.pool[:6, 0, 0] = torch.tensor(prompts[0] + prompts[1], dtype=torch.int32, device="cuda")
    dec = decode.BeamDecoder(2, 30)
    with pytest.raises(V.VsmpError, match="no page left"):
        dec.search(prompts, m, 20, stop_ids=(7, 8), pages=m.start, cache=m.cache)
    assert dec.pages.lens[:2].tolist() == [0, 0] and dec.pages.lens[2:].min() > 3
    assert dec.pages.ref.tolist() == holders(dec.pages).tolist()
    gone, _ = ctx.pages_step(dec.pages, torch.full((4,), -1, dtype=torch.int32, device="cuda"))
    assert int(gone.ref.abs().sum()) == 0


@pytest.mark.gpu
def test_the_state_of_a_search_whose_model_raised():
    """An exception of logits_fn leaves self.pages at the state that it was called with."""
    m = Recall(model(30, 3), [[1, 2, 3, 4, 5]], 3, 8, True)
    m.vocab = 30
    seen = []

    def failing(step, tokens, pages):
        seen.append(pages)
        if step == 3:
            raise KeyError("model")
        return m(step, tokens, pages)

    dec = decode.BeamDecoder(3, 30)
    with pytest.raises(KeyError):
        dec.search([[1, 2, 3, 4, 5]], failing, 8, pages=m.start, cache=m.cache)
    assert dec.pages is seen[-1] and dec.pages.lens.tolist() == [8, 8, 8]
    assert dec.pages.ref.tolist() == holders(dec.pages).tolist()
