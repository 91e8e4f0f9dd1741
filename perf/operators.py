"""The operators around the pick, as cases that can be timed and compared:

adjust    logits made ready for the pick: penalties for repeated tokens (multiplicative, presence and
          frequency), per-token biases and grammar masks
logprobs  log-probabilities and ranks of given tokens under the softmax of a row of logits
head_q4   the LM head's product with 4-bit weights and group scales

A case is a dict of plain values; `op` names the operator, the rest its sizes and types. listed() holds the
named ones, draw(rng) gives more of the same ranges. With `own` false, run() computes the operators from
elementary torch operations in 32 bits; with it true, run() calls the framework.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PENALTY = np.dtype([("repeat", "f4"), ("presence", "f4"), ("frequency", "f4"), ("window", "i4")])
INF = float("inf")


def _adjust(rows, vocab, **kw):
    """hist, prompt: the longest history and the longest part of it that is prompt; biases: the most biased tokens
    of a row; mask: none, few (a grammar that allows some 40 tokens), most (one that forbids a tenth), mixed
    (few, most, one that allows nothing, and rows without a grammar); own_penalties: the penalties are the rows' own."""
    c = dict(op="adjust", rows=rows, vocab=vocab, dtype="f32", padded=True, hist=0, prompt=0, biases=0, mask="none", own_penalties=False)
    return {**c, **kw}


def _logprobs(rows, vocab, n, **kw):
    """n: tokens asked for per row; skipped: rows among them that are not scored (id -1)."""
    return {**dict(op="logprobs", rows=rows, vocab=vocab, n=n, dtype="f32", padded=True, skipped=False), **kw}


def _head(rows, vocab, hidden, group, **kw):
    return {**dict(op="head_q4", rows=rows, vocab=vocab, hidden=hidden, group=group, zeros=False, dtype="bf16", scales="bf16"), **kw}


def listed():
    return [
        # one chat session's step: all three penalties over the last 64 tokens of a small vocabulary
        dict(_adjust(1, 49152, hist=64), name="adjust_chat_1x49152"),
        # a server's step: logits as a bf16 head leaves them, rows unpadded, every request with penalties, biases and
        # a grammar of its own or none, histories that hold the prompt
        dict(_adjust(24, 50257, dtype="bf16", padded=False, hist=2000, prompt=1500, biases=300, mask="mixed", own_penalties=True), name="adjust_serve_24x50257_bf16"),
        # structured output for a whole batch: few tokens allowed in every row
        dict(_adjust(64, 151936, hist=256, mask="few"), name="adjust_grammar_64x151936"),
        # rollouts of a large batch with long generated histories
        dict(_adjust(512, 128256, dtype="f16", hist=8192, own_penalties=True), name="adjust_rollout_512x128256_f16"),
        # one chat session: the picked token's log-probability
        dict(_logprobs(1, 49152, 1), name="logprobs_chat_1x49152"),
        # a server's step that reports the picked token and the 20 likeliest
        dict(_logprobs(32, 151936, 21), name="logprobs_top20_32x151936"),
        # a larger step on bf16 logits, rows unpadded, five alternatives
        dict(_logprobs(256, 50257, 6, dtype="bf16", padded=False), name="logprobs_serve_256x50257_bf16"),
        # the positions of prompts scored in one call, some of them left out
        dict(_logprobs(2048, 128256, 1, dtype="bf16", skipped=True), name="score_2048x128256_bf16"),
        # one token of a small model whose head is tied to its embeddings
        dict(_head(1, 49152, 576, 32), name="head_q4_1x49152x576_g32"),
        # one token of a model with a large vocabulary and a small hidden size, asymmetric groups
        dict(_head(1, 151936, 896, 32, zeros=True, scales="f16"), name="head_q4_1x151936x896_g32z"),
        # a small server batch of a model with a large hidden size, in fp16
        dict(_head(16, 128256, 4096, 128, zeros=True, dtype="f16", scales="f16"), name="head_q4_16x128256x4096_g128z_f16"),
        # a server batch of 64 rows
        dict(_head(64, 151936, 2048, 64), name="head_q4_64x151936x2048_g64"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adjust", "logprobs", "head_q4"])
    vocab = rng.choice([49152, 50257, 128256, 151936, _log_int(rng, 32000, 262144), _log_int(rng, 32000, 262144) | 1])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if op == "adjust":
        rows = min(_log_int(rng, 1, 512), 512 * 128256 // (2 * vocab))
        hist = rng.choice([0, _log_int(rng, 1, 64), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)])
        return _adjust(rows, vocab, dtype=dtype, padded=rng.random() < 0.6, hist=hist, prompt=rng.choice([0, hist // 2]),
                       biases=rng.choice([0, 0, _log_int(rng, 1, 300)]), mask=rng.choice(["none", "none", "few", "most", "mixed"]),
                       own_penalties=rng.random() < 0.5)
    if op == "logprobs":
        n = rng.choice([1, 1, 2, 6, 11, 21, rng.randint(1, 32)])
        rows = min(_log_int(rng, 1, 2048), 2048 * 128256 // (2 * vocab), max(1, 2 ** 30 // (n * vocab)))
        return _logprobs(rows, vocab, n, dtype=dtype, padded=rng.random() < 0.6, skipped=rng.random() < 0.3)
    vocab = min(vocab, 151936)
    group = rng.choice([32, 64, 128])
    hidden = group * (_log_int(rng, 512, min(4096, 64 * 4096 * 2048 // vocab)) // group)
    return _head(_log_int(rng, 1, 64), vocab, hidden, group, zeros=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "f16"]),
                 scales=rng.choice(["bf16", "f16", "f32"]))


# ---- inputs -----------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(case, seed):
    """[rows, vocab] of the case's type: a normal bulk with 16 tokens well above it, as a model's logits have."""
    g, B, V = _gen(seed), case["rows"], case["vocab"]
    x = torch.empty(B, V, device="cuda").normal_(0.0, 2.0, generator=g)
    ids = torch.randint(V // 16, (B, 16), generator=g, device="cuda") + V // 16 * torch.arange(16, device="cuda")
    x.scatter_(1, ids, 4.0 + 8.0 * torch.rand(B, 16, generator=g, device="cuda"))
    x = x.to(DTYPES[case["dtype"]])
    if case["padded"]:  # rows on 16 bytes
        p = torch.zeros(B, (V + 7) // 8 * 8, dtype=x.dtype, device="cuda")
        p[:, :V] = x
        x = p[:, :V]
    return x


def _offsets(lens):
    off = np.zeros(len(lens) + 1, np.int32)
    off[1:] = np.cumsum(lens)
    return off


def _lists(r, rows, vocab, most, likely):
    """Ragged lists of ids as (flat ids, offsets): each of a quarter of `most` to `most` ids, half of the ids among `likely`
    ones (what was said already is said again)."""
    lens = r.randint(most // 4, most + 1, size=rows)
    off = _offsets(lens)
    ids = r.randint(0, vocab, size=max(1, off[-1]))
    again = r.rand(ids.size) < 0.5
    ids[again] = likely[r.randint(0, likely.size, size=int(again.sum()))]
    return ids.astype(np.int32), off


def _masks(case, r):
    """A table of masks (bit i % 32 of word i / 32: token i is allowed) and each row's mask in it, -1 for none."""
    B, V, kind = case["rows"], case["vocab"], case["mask"]
    n = min(B, 32)
    kinds = [kind if kind != "mixed" else "empty" if m % 12 == 11 else ("few", "most")[m % 2] for m in range(n)]
    words = np.zeros((n, (V + 31) // 32), np.uint32)
    for m, k in enumerate(kinds):
        allowed = np.zeros(words.shape[1] * 32, bool)
        if k == "few":
            allowed[r.randint(0, V, size=40)] = True
        elif k == "most":
            allowed[:V] = r.rand(V) < 0.9
        words[m] = np.packbits(allowed, bitorder="little").view(np.uint32)
    row = r.randint(0, n, size=B)
    if kind == "mixed":
        row[r.rand(B) < 0.3] = -1
    return words.view(np.int32), row.astype(np.int32)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _quantised(case, seed):
    """A normal weight matrix [vocab, hidden] in groups of `group` values: two values of 4 bits a byte (the even one in
    the low half), a scale and, where the groups are asymmetric, a zero point for each group; else it is 8."""
    V, D, G = case["vocab"], case["hidden"], case["group"]
    g = _gen(seed)
    q = torch.empty(V, D // 2, dtype=torch.uint8, device="cuda")
    s = torch.empty(V, D // G, dtype=DTYPES[case["scales"]], device="cuda")
    z = torch.empty(V, D // G, dtype=torch.uint8, device="cuda") if case["zeros"] else None
    step = max(1, (1 << 26) // D)
    for a in range(0, V, step):
        w = torch.empty(min(step, V - a), D // G, G, device="cuda").normal_(0.0, 2.5 / D ** 0.5, generator=g)
        lo, hi = w.amin(2), w.amax(2)
        sc = ((hi - lo) / 15 if case["zeros"] else torch.maximum(-lo, hi) / 7).to(s.dtype)
        zp = (-lo / sc.float()).round().clamp(0, 15) if case["zeros"] else torch.full_like(lo, 8.0)
        k = ((w / sc.float()[..., None]).round() + zp[..., None]).clamp(0, 15).to(torch.uint8).reshape(-1, D)
        q[a:a + step] = k[:, 0::2] | (k[:, 1::2] << 4)
        s[a:a + step] = sc
        if z is not None:
            z[a:a + step] = zp.to(torch.uint8)
    return q, s, z


def prepare(case, seed):
    op, B, V = case["op"], case["rows"], case["vocab"]
    r = np.random.RandomState((seed + 1) & 0x7FFFFFFF)
    s = {"op": op}
    if op == "head_q4":
        s["q"], s["scales"], s["zeros"] = _quantised(case, seed)
        s["group"] = case["group"]
        x = torch.randn(B, case["hidden"], generator=_gen(seed + 1), device="cuda")
        x[:, :: case["hidden"] // 8] *= 8.0  # a few channels stand out, as they do in a model's hidden states
        s["hidden"] = x.to(DTYPES[case["dtype"]])
        return s
    s["logits"] = _logits(case, seed)
    if op == "logprobs":
        n = case["n"]
        ids = torch.randint(V, (B, n), generator=_gen(seed + 1), device="cuda")
        if n > 1:  # the picked token, then the likeliest ones
            ids[:, 1:] = s["logits"].float().topk(n - 1, dim=1).indices
        else:  # scored tokens: mostly likely ones
            top = s["logits"].float().topk(8, dim=1).indices
            pick = torch.randint(10, (B, 1), generator=_gen(seed + 2), device="cuda")
            ids = torch.where(pick < 8, top.gather(1, pick.clamp(max=7)), ids)
        if case["skipped"]:
            ids[torch.rand(B, generator=_gen(seed + 3), device="cuda") < 0.1, :] = -1
        s["ids"] = ids.to(torch.int32).contiguous()
        return s
    p = np.zeros(B if case["own_penalties"] else 1, PENALTY)
    p["repeat"], p["presence"], p["frequency"] = (a + b * r.rand(p.size).astype(np.float32) for a, b in ((1.0, 0.3), (0.0, 1.0), (0.0, 0.5)))
    p["window"] = r.choice([0, 64, 256], size=p.size) if case["own_penalties"] else 0
    s["penalty"] = _cuda(p.view(np.uint8)) if case["own_penalties"] else {f: p[f][0].item() for f in PENALTY.names}
    s["hist"] = s["hist_off"] = s["prompt_len"] = s["bias_ids"] = s["bias"] = s["bias_off"] = s["mask"] = s["mask_row"] = None
    if case["hist"]:
        likely = r.randint(0, V, size=64)
        hist, off = _lists(r, B, V, case["hist"], likely)
        s["hist"], s["hist_off"] = _cuda(hist), _cuda(off)
        if case["prompt"]:
            s["prompt_len"] = _cuda(np.minimum(r.randint(0, case["prompt"] + 1, size=B), np.diff(off)).astype(np.int32))
    if case["biases"]:
        ids, off = _lists(r, B, V, case["biases"], r.randint(0, V, size=4096))
        s["bias_ids"], s["bias_off"] = _cuda(ids), _cuda(off)
        s["bias"] = _cuda(np.where(r.rand(ids.size) < 0.1, -100.0, r.uniform(-5.0, 5.0, size=ids.size)).astype(np.float32))
    if case["mask"] != "none":
        words, row = _masks(case, r)
        s["mask"], s["mask_row"] = _cuda(words), _cuda(row)
    return s


# ---- the operators in their plain form -----------------------------------------------------------------


def _entry_rows(off, n):
    """For n entries in lists bounded by `off`: each entry's row and its place within the row."""
    at = torch.arange(n, device=off.device)
    row = torch.searchsorted(off[1:].long().contiguous(), at, right=True).clamp(max=off.numel() - 2)
    return row, at - off.long()[row]


def _plain_adjust(s):
    x = s["logits"].float()
    B, V = x.shape
    if isinstance(s["penalty"], dict):
        repeat, presence, frequency = (torch.full((B, 1), s["penalty"][f], device=x.device) for f in ("repeat", "presence", "frequency"))
        window = torch.full((B,), s["penalty"]["window"], device=x.device)
    else:
        p = s["penalty"].view(torch.float32).reshape(B, 4)
        repeat, presence, frequency = p[:, 0:1], p[:, 1:2], p[:, 2:3]
        window = s["penalty"].view(torch.int32).reshape(B, 4)[:, 3]
    y = x
    if s["hist"] is not None:
        off = s["hist_off"]
        row, at = _entry_rows(off, s["hist"].numel())
        length = (off[1:] - off[:-1]).long()
        ids = s["hist"].long()
        first = torch.where(window > 0, (length - window).clamp(min=0), 0)
        inside = (at < length[row]) & (at >= first[row]) & (ids >= 0) & (ids < V)
        cell = (row * V + ids)[inside]
        seen = torch.zeros(B * V, dtype=torch.bool, device=x.device).index_fill_(0, cell, True).reshape(B, V)
        y = torch.where(seen, torch.where(x > 0, x / repeat, x * repeat), x)
        if s["prompt_len"] is not None:
            cell = (row * V + ids)[inside & (at >= s["prompt_len"].long()[row])]
        count = torch.zeros(B * V, dtype=torch.int32, device=x.device)
        count = count.index_add_(0, cell, torch.ones_like(cell, dtype=torch.int32)).reshape(B, V)
        y = torch.where(count > 0, y - (presence + frequency * count.float()), y)
    if s["bias_ids"] is not None:
        row, at = _entry_rows(s["bias_off"], s["bias_ids"].numel())
        ids = s["bias_ids"].long()
        inside = (at < (s["bias_off"][1:] - s["bias_off"][:-1]).long()[row]) & (ids >= 0) & (ids < V)
        order = torch.arange(1, ids.numel() + 1, device=x.device, dtype=torch.int32)
        last = torch.zeros(B * V, dtype=torch.int32, device=x.device)
        last = last.scatter_reduce_(0, (row * V + ids)[inside], order[inside], "amax").reshape(B, V)
        y = torch.where(last > 0, y + s["bias"][(last - 1).clamp(min=0).long()], y)
    y = torch.where(x == -INF, x, y)
    if s["mask"] is not None:
        bit = torch.arange(V, device=x.device)
        words = s["mask"][s["mask_row"].long().clamp(min=0)]
        allowed = ((words[:, bit // 32] >> (bit % 32).int()) & 1).bool() | (s["mask_row"] < 0)[:, None]
        y = torch.where(allowed, y, -INF)
    return {"logits": y, "left": (y > -INF).sum(1).to(torch.int32)}


def _plain_logprobs(s):
    x, ids = s["logits"].float(), s["ids"].long()
    V = x.shape[1]
    top = x.amax(1, keepdim=True)
    lse = top + torch.exp(x - top).sum(1, keepdim=True).log()
    inside = (ids >= 0) & (ids < V)
    t = x.gather(1, ids.clamp(0, V - 1))
    at = torch.arange(V, device=x.device)
    before = (x[:, None, :] > t[:, :, None]) | ((x[:, None, :] == t[:, :, None]) & (at < ids[:, :, None]))
    rank = before.sum(2).to(torch.int32)
    return {"logprob": torch.where(inside, t - lse, -INF), "rank": torch.where(inside, rank, -1), "lse": lse[:, 0]}


def _plain_head(s):
    q, G = s["q"], s["group"]
    w = torch.stack((q & 15, q >> 4), 2).reshape(q.shape[0], -1, G).float()
    w = w - (s["zeros"].float()[..., None] if s["zeros"] is not None else 8.0)
    w = (w * s["scales"].float()[..., None]).reshape(q.shape[0], -1)
    return {"logits": s["hidden"].float() @ w.t()}


_ctx = None


def _context():
    """The program's sampling context, which it keeps."""
    global _ctx
    if _ctx is None:
        import verbo_amd

        _ctx = verbo_amd.Context(0)
    return _ctx


def run(s):
    op = s["op"]
    if own:
        import verbo_amd

        ctx = _context()
        if op == "adjust":
            x = s["logits"]
            pen = s["penalty"]
            if isinstance(pen, dict):
                pen = verbo_amd.Penalty(**pen)
            left = torch.empty(x.shape[0], dtype=torch.int32, device=x.device)
            y = ctx.adjust_logits(x, pen, hist=s["hist"], hist_off=s["hist_off"], prompt_len=s["prompt_len"], bias_ids=s["bias_ids"],
                                  bias=s["bias"], bias_off=s["bias_off"], mask=s["mask"], mask_row=s["mask_row"], left=left)
            return {"logits": y, "left": left}
        if op == "logprobs":
            lp, rank, lse = ctx.logprobs(s["logits"], s["ids"])
            return {"logprob": lp, "rank": rank, "lse": lse}
        return {"logits": ctx.head_logits_q4(s["hidden"], s["q"], s["scales"], s["group"], zeros=s["zeros"])}
    return {"adjust": _plain_adjust, "logprobs": _plain_logprobs, "head_q4": _plain_head}[op](s)


def work(case):
    B, V = case["rows"], case["vocab"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "head_q4":
        D, groups = case["hidden"], case["hidden"] // case["group"]
        w = V * (D // 2 + groups * (size[case["scales"]] + (1 if case["zeros"] else 0)))
        return {"bytes": w + 2 * B * D + 4 * B * V, "flops": 2 * B * V * D}
    if case["op"] == "logprobs":  # a maximum, a difference, an exponential, a sum and a comparison for each logit
        return {"bytes": B * V * size[case["dtype"]] + B * (12 * case["n"] + 4), "flops": 5 * B * V}
    masks = min(B, 32) * ((V + 31) // 32) * 4 if case["mask"] != "none" else 0
    lists = B * (4 * (case["hist"] * 5 // 8) + 8 * (case["biases"] * 5 // 8))
    return {"bytes": B * V * (size[case["dtype"]] + 4) + masks + lists + 4 * B, "flops": B * V}


# ---- the same results in 64 bits, row by row -------------------------------------------------------------


def _exact_adjust(case, s):
    x, V = s["logits"], case["vocab"]
    host = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "logits"}
    pen = host["penalty"].view(PENALTY) if "penalty" in host else None
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    left = []
    for r in range(case["rows"]):
        p = pen[r] if pen is not None else s["penalty"]
        v = x[r].double().cpu().numpy()
        y = v.copy()
        if "hist" in host:
            h = host["hist"][host["hist_off"][r]:host["hist_off"][r + 1]]
            begin = max(0, h.size - int(p["window"])) if p["window"] > 0 else 0
            said = np.unique(h[begin:])
            y[said] = np.where(v[said] > 0, v[said] / float(p["repeat"]), v[said] * float(p["repeat"]))
            made = h[max(begin, int(host["prompt_len"][r]) if "prompt_len" in host else 0):]
            ids, times = np.unique(made, return_counts=True)
            y[ids] -= float(p["presence"]) + float(p["frequency"]) * times
        if "bias_ids" in host:
            a, b = host["bias_off"][r], host["bias_off"][r + 1]
            added = dict(zip(host["bias_ids"][a:b].tolist(), host["bias"][a:b].tolist()))
            if added:
                y[list(added)] += np.array(list(added.values()))
        if "mask" in host and host["mask_row"][r] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_row"][r]].view(np.uint8), bitorder="little")[:V]
            y[bits == 0] = -np.inf
        left.append(int((y > -np.inf).sum()))
        out[r] = torch.from_numpy(y)
    return {"logits": out, "left": torch.tensor(left, dtype=torch.int32)}


def _exact_logprobs(case, s):
    lp, rank, lse = [], [], []
    for x, row in zip(s["logits"], s["ids"].tolist()):
        x = x.double()
        z = torch.logsumexp(x, 0)
        lse.append(z)
        for i in row:
            if i < 0:
                lp.append(torch.full_like(z, -INF))
                rank.append(torch.full_like(z, -1))
            else:
                lp.append(x[i] - z)
                rank.append(((x > x[i]).sum() + (x[:i] == x[i]).sum()).double())
    shape = s["ids"].shape
    return {"logprob": torch.stack(lp).reshape(shape), "rank": torch.stack(rank).reshape(shape).to(torch.int32), "lse": torch.stack(lse)}


def _exact_head(case, s):
    x, G = s["hidden"].double(), case["group"]
    out = torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device=x.device)
    step = max(1, (1 << 26) // case["hidden"])
    for a in range(0, case["vocab"], step):
        q = s["q"][a:a + step].long()
        k = torch.empty(q.shape[0], case["hidden"], dtype=torch.float64, device=x.device)
        k[:, 0::2] = (q % 16).double()
        k[:, 1::2] = (q // 16).double()
        k -= s["zeros"][a:a + step].double().repeat_interleave(G, 1) if case["zeros"] else 8
        k *= s["scales"][a:a + step].double().repeat_interleave(G, 1)
        out[:, a:a + step] = x @ k.t()
    return {"logits": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"adjust": _exact_adjust, "logprobs": _exact_logprobs, "head_q4": _exact_head}[case["op"]](case, s)
