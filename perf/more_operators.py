"""Beams and the states behind them, as cases that can be timed and compared:

select    one step of beam search: the best continuations of each group's beams over the whole vocabulary, by the
          beams' scores plus log-probabilities; stop tokens end a sequence
reorder   rows of states that follow their beams: row i takes what row parent[i] held, in place
step      one step of a cache in pages: rows take their parents' pages, grow or end; a page that is shared and about
          to be written is copied
compact   a cache in pages moved together into the lowest pages

A case is a dict of plain values; `op` names the operator, the rest its sizes and types. listed() holds the
named ones, draw(rng) gives more of the same ranges. With `own` false, run() computes the operators from
elementary torch operations; with it true, run() calls the framework.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "u8": 1}
INF = float("inf")


def _select(groups, beams, n, vocab, **kw):
    """n: beams of the next step; stops: stop tokens; idle: some groups' beams are over (their scores are -inf)."""
    return {**dict(op="select", groups=groups, beams=beams, n=n, vocab=vocab, dtype="f32", padded=True, stops=1, idle=False), **kw}


def _reorder(groups, beams, planes, heads, tokens, width, **kw):
    """planes: tensors of states, each [rows, heads, tokens, width]; ragged: rows hold fewer tokens than there is room for."""
    return {**dict(op="reorder", groups=groups, beams=beams, planes=planes, heads=heads, tokens=tokens, width=width, dtype="bf16", ragged=True), **kw}


def _pages(op, groups, beams, longest, pages, page, planes, heads, width, **kw):
    """longest: the most tokens of a row; pages of `page` tokens in the pool; each plane holds `heads` heads of `width`
    values a token, token by token or (by_head) head by head; admit: one group in 16 ends and makes room for a new prompt."""
    return {**dict(op=op, groups=groups, beams=beams, longest=longest, pages=pages, page=page, planes=planes, heads=heads, width=width,
                   dtype="bf16", by_head=False, admit=False), **kw}


def listed():
    return [
        # one chat session searched with four beams, a small vocabulary
        _select(1, 4, 4, 49152, name="select_chat_1x4x49152"),
        # the first step after the prompts: one row each becomes eight beams; logits as a bf16 head leaves them
        _select(16, 1, 8, 151936, dtype="bf16", name="select_first_16x1x151936_bf16"),
        # a server's step, rows unpadded, several stop tokens, some searches already over
        _select(24, 5, 5, 50257, dtype="f16", padded=False, stops=3, idle=True, name="select_serve_24x5x50257_f16"),
        # a large batch: 64 searches of eight beams
        _select(64, 8, 8, 128256, stops=2, name="select_batch_64x8x128256"),
        # one chat session's cache, four beams of a small model
        _reorder(1, 4, 24, 3, 512, 64, name="reorder_chat_1x4"),
        # a recurrent model's states, fp32, whole rows of an odd size
        _reorder(32, 6, 24, 1, 1, 5003, dtype="f32", ragged=False, name="reorder_state_32x6_f32"),
        # a server's caches of 16 searches, rows of different lengths
        _reorder(16, 4, 48, 2, 2048, 128, name="reorder_serve_16x4"),
        # one chat session's step over a small pool
        _pages("step", 1, 4, 512, 256, 16, 24, 2, 64, name="step_chat_1x4"),
        # a server's step without beams: rows end, prompts come in, an odd pool, head by head
        _pages("step", 256, 1, 4096, 40009, 32, 8, 4, 64, dtype="f16", by_head=True, admit=True, name="step_serve_256x1_f16"),
        # 16 searches over a model's whole cache: the shared last pages' copies count
        _pages("step", 16, 4, 2048, 2048, 64, 56, 2, 128, name="step_search_16x4"),
        # a small pool moved together
        _pages("compact", 8, 4, 512, 1024, 16, 24, 2, 64, name="compact_1024"),
        # a large pool, half of it live
        _pages("compact", 64, 2, 2048, 10007, 16, 56, 2, 128, name="compact_10007"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "reorder", "step", "compact"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "select":
        vocab = rng.choice([49152, 50257, 128256, 151936, _log_int(rng, 32000, 262144), _log_int(rng, 32000, 262144) | 1])
        n = rng.choice([1, 2, 4, 5, 8, _log_int(rng, 1, 16)])
        beams = rng.choice([1, n, n, n])
        groups = min(_log_int(rng, 1, 64), max(1, 32 * 8 * 128256 // (beams * vocab)))
        return _select(groups, beams, n, vocab, dtype=dtype, padded=rng.random() < 0.5, stops=rng.randint(0, 4), idle=rng.random() < 0.3)
    beams = rng.choice([2, 3, 4, 5, 8, _log_int(rng, 2, 16)])
    planes = 2 * _log_int(rng, 2, 28)
    if op == "reorder":
        heads, tokens, width = rng.choice([1, 2, 4, 8]), _log_int(rng, 1, 2048), rng.choice([64, 80, 128, _log_int(rng, 16, 512)])
        room = 2_000_000_000 // (planes * heads * tokens * width * SIZE[dtype])
        groups = max(1, min(_log_int(rng, 1, 48), room // beams))
        planes = max(2, min(planes, 2_000_000_000 // (groups * beams * heads * tokens * width * SIZE[dtype])))
        return _reorder(groups, beams, planes, heads, tokens, width, dtype=dtype, ragged=rng.random() < 0.7)
    page = rng.choice([8, 16, 16, 32, 64])
    longest = _log_int(rng, 4 * page, 4096 if op == "step" else 2048)
    admit = op == "step" and rng.random() < 0.5
    beams = 1 if admit and rng.random() < 0.5 else beams
    groups = _log_int(rng, 1, max(1, 256 // beams))
    pages = int(groups * (beams + 1) * (longest // page + 2) * rng.uniform(1.0, 1.6)) + 16
    heads, width = rng.choice([1, 2, 4]), rng.choice([64, 128])
    planes = max(2, min(planes, 3_000_000_000 // (pages * page * heads * width * SIZE[dtype])))
    return _pages(op, groups, beams, longest, pages, page, planes, heads, width, dtype=dtype, by_head=rng.random() < 0.4, admit=admit)


# ---- inputs -----------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rs(seed, salt):
    return np.random.RandomState((seed * 1000003 + salt) & 0x7FFFFFFF)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _filled(shape, dtype, seed):
    t = torch.empty(shape, dtype=DTYPES[dtype], device="cuda")
    return t.random_(0, 256, generator=_gen(seed)) if dtype == "u8" else t.normal_(0.0, 1.0, generator=_gen(seed))


def _parents(r, groups, beams):
    """Each row's parent among its group's rows, by the row's number in the batch: the best beams have most of the
    descendants, and one group in eight goes on as it is."""
    p = np.minimum(r.geometric(0.45, (groups, beams)) - 1, r.randint(0, beams, (groups, beams)))
    p.sort(axis=1)
    p[r.rand(groups) < 0.125] = np.arange(beams)
    return (p + beams * np.arange(groups)[:, None]).astype(np.int32)


def _prepare_select(case, seed):
    g, B, V = _gen(seed), case["groups"] * case["beams"], case["vocab"]
    # a normal bulk with 16 tokens well above it, as a model's logits have; the beams of a group agree on half of them
    x = torch.empty(B, V, device="cuda").normal_(0.0, 2.0, generator=g)
    at = V // 16 * torch.arange(16, device="cuda")
    ids = torch.randint(V // 16, (B, 16), generator=g, device="cuda") + at
    same = torch.randint(V // 16, (case["groups"], 16), generator=g, device="cuda").repeat_interleave(case["beams"], 0) + at
    ids = torch.where(torch.rand(B, 16, generator=g, device="cuda") < 0.5, ids, same)
    x.scatter_(1, ids, 4.0 + 8.0 * torch.rand(B, 16, generator=g, device="cuda"))
    x = x.to(DTYPES[case["dtype"]])
    r = _rs(seed, 1)
    stops = r.choice(V, case["stops"], replace=False).astype(int).tolist()
    for t in stops:  # a stop token is likely now and then
        x[torch.rand(B, generator=g, device="cuda") < 0.3, t] = 11.0
    if case["padded"]:  # rows on 16 bytes
        p = torch.zeros(B, (V + 7) // 8 * 8, dtype=x.dtype, device="cuda")
        p[:, :V] = x
        x = p[:, :V]
    scores = -np.sort(r.exponential(3.0, (case["groups"], case["beams"])).cumsum(1) + r.uniform(0.0, 40.0, (case["groups"], 1)), axis=1)
    if case["idle"]:
        scores[r.rand(case["groups"]) < 0.25] = -INF  # the search is over
        scores[r.rand(*scores.shape) < 0.05] = -INF  # fewer beams than there is room for
    return {"op": "select", "logits": x, "scores": _cuda(scores.astype(np.float32)), "n": case["n"], "stops": stops}


def _prepare_reorder(case, seed):
    G, W, r = case["groups"], case["beams"], _rs(seed, 2)
    states = _filled((case["planes"], G * W, case["heads"], case["tokens"], case["width"]), case["dtype"], seed)
    lens = None
    if case["ragged"]:  # the rows of a group are as long, now and then one shorter
        n = r.randint(max(1, case["tokens"] // 8), case["tokens"] + 1, size=(G, 1)).repeat(W, 1)
        lens = _cuda(np.maximum(n - (r.rand(G, W) < 0.1), 0).astype(np.int32).reshape(-1))
    return {"op": "reorder", "states": states, "parent": _cuda(_parents(r, G, W).reshape(-1)), "width": W, "lens": lens}


def _plan(case, seed):
    """The pages of a cache in use (table, lens, ref) and what the next step asks of it (parent, add). Beams share their
    prompt's pages and the first of those they made; ids are scattered over the pool."""
    r, G, W, T = _rs(seed, 3), case["groups"], case["beams"], case["page"]
    R, cap = G * W, case["longest"] // T + 2
    free = r.permutation(case["pages"]).tolist()
    table, lens, ref = np.full((R, cap), -1, np.int32), np.zeros(R, np.int32), np.zeros(case["pages"], np.int32)
    for g in range(G):
        length = int(r.randint(case["longest"] // 4, case["longest"]))
        made = int(r.randint(1, max(2, length // 4)))
        n = -(-length // T)
        if case["op"] == "compact" and r.rand() < 0.2:
            continue  # the group has ended
        first = [free.pop() for _ in range(n)]
        for b in range(W):
            apart = n if b == 0 else int(r.randint((length - made) // T, n))  # from this page on, a beam has its own
            row = first[:apart] + [free.pop() for _ in range(n - apart)]
            table[g * W + b, :n], lens[g * W + b] = row, length
            np.add.at(ref, row, 1)
    parent, add = _parents(r, G, W), np.ones((G, W), np.int32)
    add[(lens.reshape(G, W)[:, :1] == 0).repeat(W, 1)] = 0
    if case["admit"]:
        new = np.arange(G) % 16 == int(r.randint(16))
        parent[new], add[new] = -1, 0
        add[new, 0] = r.randint(1, case["longest"], int(new.sum()))
    return {"table": table, "lens": lens, "ref": ref, "parent": parent.reshape(-1), "add": add.reshape(-1)}


def _prepare_pages(case, seed):
    s = {k: _cuda(v) for k, v in _plan(case, seed).items()}
    inner = (case["heads"], case["page"], case["width"]) if case["by_head"] else (case["page"], case["heads"], case["width"])
    s.update(op=case["op"], page=case["page"], by_head=case["by_head"], cache=_filled((case["planes"], case["pages"]) + inner, case["dtype"], seed))
    return s


def prepare(case, seed):
    return {"select": _prepare_select, "reorder": _prepare_reorder, "step": _prepare_pages, "compact": _prepare_pages}[case["op"]](case, seed)


# ---- the operators in their plain form -----------------------------------------------------------------


def _places(first, take, width):
    """For the flags `take` [G, n]: where each is to be put among `width` places (those after the last go to one more)."""
    at = take.long().cumsum(1) - 1
    return torch.where(take & (at < width) & first, at, width)


def _plain_select(s):
    x, scores, N = s["logits"].float(), s["scores"].double(), s["n"]
    G, W = scores.shape
    B, V = x.shape
    d = x.double()
    top = d.amax(1, keepdim=True)
    lse = top + torch.exp(d - top).sum(1, keepdim=True).log()
    live = torch.isfinite(lse) & torch.isfinite(scores.reshape(B, 1))
    # a row's order as whole numbers: the value, then the lowest token
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = bits * V + (V - 1 - torch.arange(V, device=x.device))
    none = -(1 << 62)
    key = torch.where(x > -INF, key, none)
    stops = torch.tensor(s["stops"], dtype=torch.long, device=x.device)
    ends = key[:, stops]
    key[:, stops] = none
    key = torch.cat((key.topk(min(N, V), 1).values, ends), 1)
    is_end = torch.arange(key.shape[1], device=x.device) >= min(N, V)
    key, order = key.sort(dim=1, descending=True, stable=True)
    is_end = is_end[order].reshape(G, -1)
    token = V - 1 - key.remainder(V)
    there = (key > none) & live
    score = torch.where(there, scores.reshape(B, 1) + (d.gather(1, token) - lse), -INF).reshape(G, -1)
    row = torch.arange(B, device=x.device)[:, None].expand(B, key.shape[1]).reshape(G, -1)
    score, order = score.sort(dim=1, descending=True, stable=True)
    token, row, is_end = (t.reshape(G, -1).gather(1, order) for t in (token, row, is_end))
    there = score > -INF
    own_row = torch.arange(G, device=x.device)[:, None] * W + torch.arange(N + 1, device=x.device) % W
    early = torch.arange(score.shape[1], device=x.device) < N

    def gathered(at):
        return (torch.full((G, N + 1), -1, device=x.device).scatter_(1, at, token)[:, :N].to(torch.int32),
                own_row.clone().scatter_(1, at, row)[:, :N].to(torch.int32),
                torch.full((G, N + 1), -INF, dtype=torch.float64, device=x.device).scatter_(1, at, score)[:, :N].float())

    token_, parent_, score_ = gathered(_places(there, there & ~is_end, N))
    end = there & is_end & early
    end_token, end_parent, end_score = gathered(_places(there, end, N))
    return {"token": token_, "parent": parent_, "score": score_, "end_token": end_token, "end_parent": end_parent, "end_score": end_score,
            "n_end": end.sum(1).to(torch.int32)}


def _plain_reorder(s):
    x = s["states"]
    taken = x[:, s["parent"].long()]
    if s["lens"] is not None:
        held = torch.arange(x.shape[3], device=x.device) < s["lens"][s["parent"].long()][:, None]
        taken = torch.where(held[None, :, None, :, None], taken, x)
    x.copy_(taken)
    return {"states": x}


def _plain_step(s):
    table, lens, ref, T = s["table"].long(), s["lens"].long(), s["ref"].long(), s["page"]
    parent, add = s["parent"].long(), s["add"].long()
    R, cap = table.shape
    P, dev = ref.numel(), table.device
    j = torch.arange(cap, device=dev)
    row = torch.arange(R, device=dev)
    length = torch.where(parent >= 0, lens[parent.clamp(min=0)], 0)
    wanted = (length + add).clamp(min=0)
    fits = wanted <= cap * T
    wanted = torch.where(fits, wanted, length)
    have, want = (length + T - 1) // T, (wanted + T - 1) // T
    old = torch.where(j < ((lens + T - 1) // T)[:, None], table, P)
    new = torch.where(j < torch.minimum(have, want)[:, None], table[parent.clamp(min=0)], P)
    held = torch.zeros(P + 1, dtype=torch.long, device=dev).index_add_(0, new.reshape(-1), torch.ones_like(new).reshape(-1))
    held.index_add_(0, old.reshape(-1), -torch.ones_like(old).reshape(-1))
    ref = ref + held[:P]
    # the last page of a row that grows: copied, unless all that hold it grow in it and this one is the longest of them
    grows = wanted > length
    part = length % T
    into = grows & (part > 0)
    last = torch.where(into, new.gather(1, (length // T).clamp(max=cap - 1)[:, None])[:, 0], P)
    writers = torch.zeros(P + 1, dtype=torch.long, device=dev).index_add_(0, last, torch.ones_like(last))
    order = length * R + (R - 1 - row)
    longest = torch.zeros(P + 1, dtype=torch.long, device=dev).scatter_reduce_(0, last, order, "amax")
    copied = into & ((torch.cat((ref, ref[:1]))[last] != writers[last]) | (longest[last] != order))
    need = torch.where(grows, want - have + copied.long(), 0)
    end = need.cumsum(0)
    is_free = ref <= 0
    fits &= (need == 0) | (end <= is_free.sum())
    free = torch.argsort((~is_free).to(torch.int8), stable=True)
    copied &= fits
    need = torch.where(fits, need, 0)
    wanted = torch.where(fits, wanted, length)
    k = j - (have - copied.long())[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    got = free[(end[:, None] - need[:, None] + k).clamp(0, P - 1)]
    new = torch.where(fresh, got, new)
    ref = torch.cat((ref, ref[:1])).index_add_(0, torch.where(copied, last, P), -torch.ones_like(last))
    ref.index_fill_(0, torch.where(fresh, got, P).reshape(-1), 1)
    # the copies
    x = s["cache"]
    who = copied.nonzero()[:, 0]
    src, dst = last[who], new[who, length[who] // T]
    t = torch.arange(T, device=dev) < part[who][:, None]
    t = t[None, :, None, :, None] if s["by_head"] else t[None, :, :, None, None]
    x[:, dst] = torch.where(t, x[:, src], x[:, dst])
    new = torch.where(new == P, -1, new)
    return {"table": new.to(torch.int32), "lens": wanted.to(torch.int32), "ref": ref[:P].to(torch.int32), "ok": fits.to(torch.int32), "cache": x}


def _plain_compact(s):
    table, lens, ref, T = s["table"].long(), s["lens"], s["ref"], s["page"]
    P, dev = ref.numel(), table.device
    live = ref > 0
    n = live.sum()
    page = torch.arange(P, device=dev)
    moves, room = live & (page >= n), ~live & (page < n)
    src, dst = moves.nonzero()[:, 0], room.nonzero()[:, 0]
    moved = torch.where(live, page, -1)
    moved[src] = dst
    x = s["cache"]
    x[:, dst] = x[:, src]
    used = torch.arange(table.shape[1], device=dev) < ((lens + T - 1) // T)[:, None]
    new_ref = torch.where(page < n, ref, 0)
    new_ref[dst] = ref[src]
    return {"table": torch.where(used, moved[table.clamp(min=0)], -1).to(torch.int32), "lens": lens.clone(), "ref": new_ref.to(torch.int32),
            "moved": moved.to(torch.int32), "live": n.to(torch.int32).reshape(1), "cache": x}


_ctx = None


def _context():
    """The program's sampling context, which it keeps."""
    global _ctx
    if _ctx is None:
        import verbo_amd

        _ctx = verbo_amd.Context(0)
    return _ctx


def _handles(s):
    """What a program makes of its caches once and keeps: their planes, the pages in use and the next step's."""
    if "kept" not in s:
        import verbo_amd

        if s["op"] == "reorder":
            s["kept"] = verbo_amd.Planes(s["states"].unbind(0), token_dim=2)
        else:
            pages = verbo_amd.Pages(s["table"], s["lens"], s["ref"], s["page"])
            s["kept"] = verbo_amd.Planes(s["cache"].unbind(0), token_dim=2 if s["by_head"] else 1), pages, pages.like()
    return s["kept"]


def run(s):
    op = s["op"]
    if own:
        ctx = _context()
        if op == "select":
            return ctx.beam_select(s["logits"], s["scores"], s["n"], stop_ids=s["stops"])._asdict()
        if op == "reorder":
            ctx.reorder_rows(_handles(s), s["parent"], s["width"], lens=s["lens"])
            return {"states": s["states"]}
        planes, pages, to = _handles(s)
        if op == "step":
            to, ok = ctx.pages_step(pages, parent=s["parent"], add=s["add"], cache=planes, out=to)
            return {"table": to.table, "lens": to.lens, "ref": to.ref, "ok": ok, "cache": s["cache"]}
        to, moved, live = ctx.pages_compact(pages, cache=planes, out=to)
        return {"table": to.table, "lens": to.lens, "ref": to.ref, "moved": moved, "live": live, "cache": s["cache"]}
    return {"select": _plain_select, "reorder": _plain_reorder, "step": _plain_step, "compact": _plain_compact}[op](s)


def work(case):
    if case["op"] == "select":  # a maximum, a difference, an exponential, a sum and a comparison for each logit
        B = case["groups"] * case["beams"]
        live = 0.72 if case["idle"] else 1.0
        return {"bytes": live * B * case["vocab"] * SIZE[case["dtype"]] + 4 * B + case["groups"] * (24 * case["n"] + 4), "flops": 5 * live * B * case["vocab"]}
    if case["op"] == "reorder":  # a row that has another parent is written, each such parent read once
        r = _rs(0, 2)
        n = np.full((case["groups"], 1), case["tokens"])
        if case["ragged"]:
            n = r.randint(max(1, case["tokens"] // 8), case["tokens"] + 1, size=(case["groups"], 1))
            r.rand(case["groups"], case["beams"])
        p = _parents(r, case["groups"], case["beams"])
        at = np.arange(p.size).reshape(p.shape)
        rows = [int(m) * (int((q != i).sum()) + len(set(q[q != i].tolist()))) for m, q, i in zip(n[:, 0], p, at)]
        return {"bytes": sum(rows) * case["planes"] * case["heads"] * case["width"] * SIZE[case["dtype"]] + 4 * p.size, "flops": 0}
    p, T = _plan(case, 0), case["page"]
    page = case["planes"] * case["heads"] * case["width"] * SIZE[case["dtype"]]  # bytes of a token
    used = -(-p["lens"] // T)
    tables = 4 * int(used.sum()) + 4 * p["table"].size + 8 * case["pages"] + 16 * used.size
    if case["op"] == "compact":
        live = p["ref"] > 0
        return {"bytes": 2 * page * T * int(live[int(live.sum()):].sum()) + tables + 4 * case["pages"], "flops": 0}
    copied = 0
    seen = set()
    for i in np.flatnonzero((p["parent"] >= 0) & (p["add"] > 0)):
        length = int(p["lens"][p["parent"][i]])
        if length % T:
            q = int(p["table"][p["parent"][i], length // T])
            copied += length % T if q in seen else 0
            seen.add(q)
    return {"bytes": 2 * page * copied + tables, "flops": 0}


# ---- the same results from the definitions, group by group and row by row --------------------------------


def _exact_select(case, s):
    x, N, W = s["logits"], s["n"], case["beams"]
    out = {k: [] for k in ("token", "parent", "score", "end_token", "end_parent", "end_score", "n_end")}
    for g, scores in enumerate(s["scores"].double().cpu().numpy()):
        found = []
        for b in range(W):
            v = x[g * W + b].double()
            z = torch.logsumexp(v, 0)
            if np.isfinite(scores[b]) and torch.isfinite(z):
                few = v.topk(min(N + len(s["stops"]), v.numel())).values[-1]
                at = torch.cat((torch.nonzero((v >= few) & (v > -INF))[:, 0], torch.tensor(s["stops"], dtype=torch.long, device=v.device))).unique()
                found += [(-(scores[b] + a), b, -c, t) for a, c, t in zip((v[at] - z).tolist(), v[at].tolist(), at.tolist()) if c > -INF]
        found.sort()
        ends = [(t, g * W + b, -a) for a, b, _, t in found[:N] if t in s["stops"]]
        goes = [(t, g * W + b, -a) for a, b, _, t in found if t not in s["stops"]][:N]
        for name, rows in (("", goes), ("end_", ends)):
            rows = rows + [(-1, g * W + i % W, -INF) for i in range(len(rows), N)]
            for k, v in zip(("token", "parent", "score"), zip(*rows)):
                out[name + k].append(v)
        out["n_end"].append(len(ends))
    return {k: torch.tensor(v, dtype=torch.float64 if "score" in k else torch.int32) for k, v in out.items()}


def _exact_reorder(case, s):
    x, parent = s["states"], s["parent"].tolist()
    was = x.clone()
    for i, p in enumerate(parent):
        n = x.shape[3] if s["lens"] is None else int(s["lens"][p])
        if p != i:
            x[:, i, :, :n] = was[:, p, :, :n]
    return {"states": x}


def _copy_page(s, src, dst, tokens):
    x = s["cache"]
    if s["by_head"]:
        x[:, dst, :, :tokens] = x[:, src, :, :tokens]
    else:
        x[:, dst, :tokens] = x[:, src, :tokens]


def _exact_step(case, s):
    T, P = case["page"], case["pages"]
    table, lens, parent, add = (s[k].cpu().numpy() for k in ("table", "lens", "parent", "add"))
    cap = table.shape[1]
    rows, ref = [], s["ref"].cpu().numpy().astype(np.int64)
    for i in range(len(lens)):
        ref[table[i, :-(-lens[i] // T)]] -= 1
    for i, p in enumerate(parent):
        n = int(lens[p]) if p >= 0 else 0
        to = max(0, n + int(add[i]))
        rows.append([table[p, :-(-min(n, to if to <= cap * T else n) // T)].tolist() if p >= 0 else [], n, to if to <= cap * T else n, to <= cap * T])
        np.add.at(ref, rows[-1][0], 1)
    users = {}  # of a page that is begun: the rows that grow in it
    for i, (pages, n, to, ok) in enumerate(rows):
        if to > n and n % T:
            users.setdefault(pages[-1], []).append(i)
    keeps = {q: max(w, key=lambda i: (rows[i][1], -i)) for q, w in users.items() if len(w) == ref[q]}
    free = np.flatnonzero(ref <= 0).tolist()
    asked = 0
    for i, (pages, n, to, ok) in enumerate(rows):
        if to <= n:
            continue
        away = n % T > 0 and keeps.get(pages[-1]) != i
        need = -(-to // T) - -(-n // T) + away
        asked += need
        if need and asked > len(free):
            rows[i][2:] = n, False
            continue
        got = free[asked - need:asked]
        ref[got] = 1
        if away:
            _copy_page(s, pages[-1], got[0], n % T)
            ref[pages.pop()] -= 1
        pages += got
    out = np.full(table.shape, -1, np.int32)
    for i, r in enumerate(rows):
        out[i, :len(r[0])] = r[0]
    t = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32)  # noqa: E731
    return {"table": t(out), "lens": t([r[2] for r in rows]), "ref": t(ref), "ok": t([int(r[3]) for r in rows]), "cache": s["cache"]}


def _exact_compact(case, s):
    table, lens, ref = (s[k].cpu().numpy() for k in ("table", "lens", "ref"))
    live = [p for p in range(case["pages"]) if ref[p] > 0]
    holes = [p for p in range(len(live)) if ref[p] <= 0]
    to = {p: p for p in live}
    to.update(zip([p for p in live if p >= len(live)], holes))
    for a, b in to.items():
        if a != b:
            _copy_page(s, a, b, case["page"])
    out, new, moved = np.full(table.shape, -1, np.int32), np.zeros_like(ref), np.full(ref.shape, -1, np.int32)
    for i, n in enumerate(lens):
        for k in range(-(-int(n) // case["page"])):
            out[i, k] = to[int(table[i, k])]
    for a, b in to.items():
        new[b], moved[a] = ref[a], b
    t = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32)  # noqa: E731
    return {"table": t(out), "lens": t(lens), "ref": t(new), "moved": t(moved), "live": t([len(live)]), "cache": s["cache"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "step": _exact_step, "compact": _exact_compact}[case["op"]](case, s)
