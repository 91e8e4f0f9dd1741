"""Batched decoding on the GPU: N sequences picked together, each with its own sampling options,
their draw streams and history windows on the device (vsmp_bsampler in include/vsmp.h).

The reference serves one request at a time (cli/serve.cpp:168) and binds one verbo_generate per
session (python/verbo/__init__.py:206-236). Here a continuous-batching step picks for every live
sequence at once from [N x V] device logits: per sequence the semantics are those of
verbo::generate's loop (reference src/sampler.cpp:111-181) — the prompt is accepted into the
history, a stop id ends the sequence without being accepted, every other id is accepted and
counted until max_tokens. Only the N picked ids come back to the host each step, for the stop
check; the accepts happen on the device.

    dec = BatchDecoder([Opts(max_tokens=64, temp=0.8, seed=1), Opts(temp=0.0)], vocab=V)
    toks = dec.generate(prompts, logits_fn, stop_ids={2})   # logits_fn(step, last, live) -> cuda [N, V]

A server keeps a decoder of a fixed number of slots and lets requests take them as they arrive and
free them as they finish (continuous batching); each step samples only the live slots:

    dec = BatchDecoder.with_slots(8, vocab=V)
    res = dec.serve([Request(prompt, Opts(max_tokens=32, seed=7), arrival=3), ...], logits_fn, stop_ids={2})
    # logits_fn(reqs, steps, last) -> cuda [len(reqs), V]: each live request's next position

Beam search keeps `width` beams of every prompt, and lets the states behind them follow (include/vsmp_beam.h):

    res = BeamDecoder(4, vocab=V).search(prompts, logits_fn, max_tokens=64, stop_ids={2}, pages=pages, cache=planes)
    # logits_fn(step, tokens, pages) -> cuda [rows, V]; res[j]: the prompt's sequences as (ids, score), the best first

`Opts` mirrors the reference's option block (`_Opts`, python/verbo/__init__.py:16-25, the C ABI's
verbo_gen_opts): the fields verbo_generate lets a caller set. Like verbo_generate, which keeps the
model's repeat_last (src/capi.cpp:131-151), BatchDecoder takes repeat_last (default 64) apart.
"""
import ctypes

import numpy as np

from . import Context, Params, Penalty, VsmpError, _adjust_args, _err, _penalty_rows, load_library, to_device_penalties

__all__ = ["Opts", "Request", "BatchDecoder", "BeamDecoder", "params_of"]


class Opts(ctypes.Structure):
    """verbo_gen_opts (reference include/verbo/verbo.h; python/verbo/__init__.py:16-25 `_Opts`)."""

    _fields_ = [
        ("max_tokens", ctypes.c_int),
        ("temp", ctypes.c_float),
        ("top_k", ctypes.c_int),
        ("top_p", ctypes.c_float),
        ("min_p", ctypes.c_float),
        ("repeat", ctypes.c_float),
        ("seed", ctypes.c_ulonglong),
    ]

    def __init__(self, max_tokens=256, temp=0.7, top_k=40, top_p=0.9, min_p=0.0, repeat=1.0, seed=0):
        super().__init__(max_tokens, temp, top_k, top_p, min_p, repeat, seed)


class Request:
    """One generation request of a serving loop: the prompt's ids, its options (Opts), the window
    of its repetition penalty and the step at which it arrives. penalty: None, or a Penalty taken from its
    logits before each pick, over the last ids of the prompt and the answer: penalty.window of them, at most
    repeat_last (each: all, where it is 0 or less). prompt_len: how many ids at the prompt's start count for the
    penalty's `repeat` alone, not for presence and frequency (len(prompt) leaves the prompt out of those)."""

    def __init__(self, prompt, opts, repeat_last=64, arrival=0, penalty=None, prompt_len=0):
        self.prompt = np.ascontiguousarray(prompt, dtype=np.int32)
        self.opts = opts
        self.repeat_last = int(repeat_last)
        self.arrival = int(arrival)
        self.penalty = penalty
        if penalty is not None:
            _penalty_rows([penalty])  # refused here, not in the middle of a loop that serves others too
        self.prompt_len = int(prompt_len)
        if not 0 <= self.prompt_len <= self.prompt.size:
            raise VsmpError("need 0 <= prompt_len <= the prompt's ids")


def params_of(o, repeat_last=64):
    """The verbo::Sampling that verbo_generate builds from an option block (src/capi.cpp:136-146)."""
    return Params(o.temp, o.top_k, o.top_p, o.min_p, o.repeat, repeat_last, o.seed)


_sig_done = False


def _lib():
    global _sig_done
    lib = load_library()
    if not _sig_done:
        P = ctypes.c_void_p
        for name, (res, args) in {
            "vsmp_bsampler_new": (P, [ctypes.c_int, ctypes.c_int, P, ctypes.c_int]),
            "vsmp_bsampler_free": (None, [P]),
            "vsmp_bsampler_accept_host": (ctypes.c_int, [P, ctypes.c_int, P, ctypes.c_int]),
            "vsmp_bsampler_pick": (ctypes.c_int, [P, P, ctypes.c_int, ctypes.c_longlong, P, P]),
            "vsmp_bsampler_accept": (ctypes.c_int, [P, P, P, P]),
            "vsmp_bsampler_full": (ctypes.c_int, [P, P]),
            "vsmp_bsampler_admit": (ctypes.c_int, [P, ctypes.c_int, P, P, ctypes.c_int, P]),
            "vsmp_bsampler_pick_rows": (ctypes.c_int, [P, P, ctypes.c_int, ctypes.c_longlong, P, ctypes.c_int, P, P]),
            "vsmp_bsampler_accept_rows": (ctypes.c_int, [P, P, P, P, ctypes.c_int, P]),
            "vsmp_bsampler_adjust_rows": (ctypes.c_int, [P, P, ctypes.c_int, ctypes.c_longlong, ctypes.c_int, P, ctypes.c_int,
                                                         P, ctypes.c_int, P, P, P, P, P, ctypes.c_longlong, ctypes.c_int, P, P,
                                                         ctypes.c_longlong, P, P]),
        }.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _sig_done = True
    return lib


class BatchDecoder:
    """N sequences decoded together on one device (vsmp_bsampler).

    opts: one Opts per sequence. cap: history ids each sequence may hold (at least 4 * repeat_last;
    default: that, or, with repeat_last <= 0, the longest prompt plus max_tokens must fit)."""

    def __init__(self, opts, vocab, repeat_last=64, cap=None, device=0):
        self.lib = _lib()
        self.opts = list(opts)
        self.n = len(self.opts)
        self.vocab = int(vocab)
        self.device = device
        rl = repeat_last if np.ndim(repeat_last) else [repeat_last] * self.n
        self.params = (Params * self.n)(*[params_of(o, int(r)) for o, r in zip(self.opts, rl)])
        need = max([4 * int(r) for r in rl if int(r) > 0] + [1])
        self.cap = int(cap) if cap is not None else max(need, 4096)
        self._h = self.lib.vsmp_bsampler_new(int(device), self.n, ctypes.cast(self.params, ctypes.c_void_p), self.cap)
        if not self._h:
            raise _err()

    def close(self):
        if getattr(self, "_h", None):
            self.lib.vsmp_bsampler_free(self._h)
            self._h = None

    def __del__(self):
        self.close()

    def accept_prompt(self, row, ids):
        a = np.ascontiguousarray(ids, dtype=np.int32)
        if self.lib.vsmp_bsampler_accept_host(self._h, int(row), a.ctypes.data_as(ctypes.c_void_p) if a.size else None,
                                             int(a.size)) != 0:
            raise _err()

    def pick(self, logits, out, stream):
        """One pick per sequence from device logits [N, V] (rows may be strided) into device out[N]."""
        if logits.shape != (self.n, self.vocab) or logits.stride(1) != 1:
            raise VsmpError("logits must be a [N, V] device tensor with contiguous rows")
        if self.lib.vsmp_bsampler_pick(self._h, logits.data_ptr(), self.vocab, logits.stride(0), out.data_ptr(),
                                       ctypes.c_void_p(stream.cuda_stream)) != 0:
            raise _err()

    def accept(self, ids, live, stream):
        """Sampler::accept of ids[r] for every row with live[r] != 0 (device int32 tensors)."""
        if self.lib.vsmp_bsampler_accept(self._h, ids.data_ptr(), live.data_ptr(),
                                         ctypes.c_void_p(stream.cuda_stream)) != 0:
            raise _err()

    def generate(self, prompts, logits_fn, stop_ids=()):
        """Decodes every sequence to its end: per step, logits_fn(step, last, live) returns the device
        logits [N, V] of the next position of every row (last: each row's last id, or -1 before its
        first pick; live: which rows still decode, a host bool array). Returns per row (tokens,
        stopped): the ids generated and whether a stop id ended the sequence. Sequence r decodes in
        slot r with the options given at construction; each step samples the live rows only (serve()
        with every request arriving at step 0)."""
        import torch

        rl = [int(p.repeat_last) for p in self.params]
        reqs = [Request(p, o, r, 0) for p, o, r in zip(prompts, self.opts, rl)]
        n = self.n

        def rows_of(js, steps, last):
            # every live sequence was admitted at step 0 and picked at every step since: one step for all
            last_all = np.full(n, -1, np.int64)
            last_all[js] = last
            live = np.zeros(n, bool)
            live[js] = True
            lg = logits_fn(int(steps[0]), last_all, live)
            return lg.index_select(0, torch.as_tensor(js, dtype=torch.long, device=lg.device))

        return self.serve(reqs, rows_of, stop_ids)

    @classmethod
    def with_slots(cls, slots, vocab, cap=4096, device=0):
        """A decoder of `slots` slots for serve(): every slot free until a request takes it.
        cap: history ids a slot holds (at least 4 * repeat_last of every request admitted)."""
        return cls([Opts(max_tokens=0, temp=0.0)] * int(slots), vocab, repeat_last=0, cap=cap, device=device)

    def admit(self, slot, params, prompt, stream):
        """vsmp_bsampler_admit: a new sequence (verbo::Sampler(params) that accepted `prompt`) takes
        `slot`, ordered on `stream` after the slot's earlier work."""
        a = np.ascontiguousarray(prompt, dtype=np.int32)
        if self.lib.vsmp_bsampler_admit(self._h, int(slot), ctypes.byref(params), a.ctypes.data if a.size else None,
                                        int(a.size), ctypes.c_void_p(stream.cuda_stream)) != 0:
            raise _err()

    def pick_rows(self, logits, rows, out, stream):
        """One pick for each live slot rows[i] (device int32) from device logits [len(rows), V]."""
        n = int(rows.numel())
        if logits.shape != (n, self.vocab) or logits.stride(1) != 1:
            raise VsmpError("logits must be a [len(rows), V] device tensor with contiguous rows")
        if self.lib.vsmp_bsampler_pick_rows(self._h, logits.data_ptr(), self.vocab, logits.stride(0), rows.data_ptr(), n,
                                            out.data_ptr(), ctypes.c_void_p(stream.cuda_stream)) != 0:
            raise _err()

    def adjust_rows(self, logits, rows, penalty=None, prompt_len=None, bias_ids=None, bias=None, bias_off=None, mask=None,
                    mask_row=None, out=None, left=None, stream=None):
        """Context.adjust_logits for the live slots rows[i] (device int32, distinct), before pick_rows: row i is
        penalised by slot rows[i]'s history. Per-row arrays go by row of the call. A window is at most the slot's
        repeat_last where that is above 0 (and that for a window of 0); prompt_len counts from the sequence's first
        id, also after the slot has dropped it. Returns the adjusted logits (`out`)."""
        dev = logits.device
        if dev.type != "cuda" or dev.index != self.device or tuple(logits.shape) != (rows.numel(), self.vocab):
            raise VsmpError("logits must be a [len(rows), V] tensor on the decoder's device")
        if rows.dtype.itemsize != 4 or rows.is_floating_point() or rows.device != dev or not rows.is_contiguous():
            raise VsmpError("rows must be a contiguous int32 tensor on the decoder's device")
        x, (n, vocab), pen, _, rest, out = _adjust_args(logits, penalty, None, None, prompt_len, bias_ids, bias, bias_off,
                                                        mask, mask_row, out, left, stream, csr=False)
        if self.lib.vsmp_bsampler_adjust_rows(self._h, *x, vocab, rows.data_ptr(), n, *pen, *rest) != 0:
            raise _err()
        return out

    def accept_rows(self, ids, rows, active, stream):
        """Sampler::accept of ids[i] into slot rows[i] where active[i] != 0 (device int32 tensors)."""
        if self.lib.vsmp_bsampler_accept_rows(self._h, ids.data_ptr(), rows.data_ptr(), active.data_ptr(),
                                              int(rows.numel()), ctypes.c_void_p(stream.cuda_stream)) != 0:
            raise _err()

    def serve(self, requests, logits_fn, stop_ids=()):
        """Continuous batching over the decoder's slots: each step, requests that have arrived take
        free slots (in arrival order, the lowest slot first), then every live slot is sampled at once
        and only the live slots: logits_fn(reqs, steps, last) returns the device logits
        [len(reqs), V] of the requests reqs (indices into `requests`) at their own steps `steps`
        after their last ids `last` (-1 before a request's first pick). Per request, the semantics
        are those of verbo::generate (reference src/sampler.cpp:111-181; cli/serve.cpp:139-192 runs
        it per request): the prompt accepted first, a stop id ends the sequence unaccepted, any other
        id is accepted and counted until max_tokens. A finished request's slot is free for the next
        step. Returns per request (tokens, stopped); self.schedule holds per step the (request,
        slot) pairs that were sampled."""
        import torch

        stops = set(int(x) for x in stop_ids)
        dev = torch.device("cuda", self.device)
        stream = torch.cuda.current_stream(dev)
        out = torch.empty(self.n, dtype=torch.int32, device=dev)
        order = sorted(range(len(requests)), key=lambda j: (requests[j].arrival, j))
        queue = list(order)
        free = list(range(self.n))
        live = {}  # slot -> request
        toks = [[] for _ in requests]
        stopped = [False] * len(requests)
        steps = [0] * len(requests)
        last = [-1] * len(requests)
        held, pens, own = None, None, None  # the requests, penalties and prompt lengths that are on the device
        self.schedule = []
        step = 0
        while queue or live:
            while queue and requests[queue[0]].arrival <= step and free:
                j = queue.pop(0)
                r = requests[j]
                if r.opts.max_tokens <= 0:
                    continue  # nothing to generate: done without a slot
                slot = free.pop(0)
                self.admit(slot, params_of(r.opts, r.repeat_last), r.prompt, stream)
                live[slot] = j
            if not live:
                step += 1
                continue
            slots = sorted(live)
            reqs = [live[s] for s in slots]
            rows = torch.tensor(slots, dtype=torch.int32, device=dev)
            lg = logits_fn(reqs, [steps[j] for j in reqs], [last[j] for j in reqs])
            if any(requests[j].penalty is not None for j in reqs):
                now = _penalty_rows([requests[j].penalty or Penalty() for j in reqs])
                lens = [requests[j].prompt_len for j in reqs]
                if (reqs, now.tobytes(), lens) != held:  # by value: a caller may change a request as it goes
                    pens, own = to_device_penalties(now, dev), torch.tensor(lens, dtype=torch.int32, device=dev)
                    held = reqs, now.tobytes(), lens
                lg = self.adjust_rows(lg, rows, pens, prompt_len=own, stream=stream)
            self.pick_rows(lg, rows, out[:len(slots)], stream)
            self.schedule.append(list(zip(reqs, slots)))
            ids = out[:len(slots)].cpu().numpy()  # the only per-step copy to the host: one id per live slot
            take = np.zeros(len(slots), np.int32)
            done = []
            for i, (s, j) in enumerate(zip(slots, reqs)):
                t = int(ids[i])
                steps[j] += 1
                if t in stops:  # not accepted, not counted (src/sampler.cpp:159-162)
                    stopped[j] = True
                    done.append(s)
                    continue
                take[i] = 1
                toks[j].append(t)
                last[j] = t
                if len(toks[j]) >= requests[j].opts.max_tokens:
                    done.append(s)
            self.accept_rows(out[:len(slots)], rows, torch.from_numpy(take).to(dev), stream)
            for s in done:
                del live[s]
                free.append(s)
            free.sort()
            step += 1
        if self.lib.vsmp_bsampler_full(self._h, ctypes.c_void_p(stream.cuda_stream)) != 0:
            raise VsmpError("a sequence's history outgrew its slot's region (cap)")
        return list(zip(toks, stopped))


class BeamDecoder:
    """Beam search on one device: `width` beams of each prompt, selected by Context.beam_select, with caches in pages
    (Context.pages_step) or states held row by row (Context.reorder_rows) that follow them. The reference has no
    such search; a greedy one (width 1) picks the tokens that its sampler picks at temp 0 (src/sampler.cpp:66-70)."""

    def __init__(self, width, vocab, device=0):
        self.width, self.vocab, self.device = int(width), int(vocab), int(device)
        if not 1 <= self.width <= 64 or self.vocab < 1:
            raise VsmpError("need 1 <= width <= 64 and a vocabulary")
        self.ctx = Context(self.device)

    def search(self, prompts, logits_fn, max_tokens, stop_ids=(), length_penalty=1.0, pages=None, cache=None, states=None):
        """For each prompt the best `width` sequences, the best first, as (ids, score): the generated ids (a stop id ends a
        sequence and is not among them) and their log-probabilities' sum divided by length ** length_penalty, the
        length counting the stop id. A search ends when it has `width` ended sequences of which none is behind what its
        best beam would score if it ended now, when no beam is left, or at max_tokens, where the beams count as they are.

        logits_fn(step, tokens, pages) returns device logits [rows, V]. Step 0: a row for each prompt (tokens None); then a
        row for each beam, width of a prompt one after the other, tokens (device int32 [rows]) their last ids, -1 for
        a beam that is not live (its logits are not read). pages: None, or a Pages with a row for each prompt, which
        holds the prompt's tokens; logits_fn gets the state in which each beam has room for its last id. cache: the
        Planes whose rows are the pages, as Context.pages_step takes them. states: None, or a Planes of len(prompts) *
        width rows in which row j * width holds prompt j's state when the search begins (its tokens, where the planes
        have a token_dim); the rows follow their beams after every step. self.pages: the state that the search
        ended with, all its rows given up. Where the search raises (no page left, or out of logits_fn), it is the state
        that the last step left, whose rows hold their pages until the caller gives them up; `pages` is not to be
        used again: pages of its prompts may have been given up and written by other beams."""
        import torch

        dev = torch.device("cuda", self.device)
        G, W, ctx = len(prompts), self.width, self.ctx
        stops = sorted(set(int(t) for t in stop_ids))
        self.pages = pages
        if G == 0 or max_tokens <= 0:
            return [[] for _ in prompts]
        if pages is not None and pages.lens.numel() != G:
            raise VsmpError("pages must have a row for each prompt")
        if states is not None and states.rows != G * W:
            raise VsmpError("states must have width rows for each prompt")
        held = None
        if states is not None and states.token_dim is not None:
            held = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev).repeat_interleave(W)
        scores = torch.zeros(G, 1, device=dev)
        tokens = None
        back = []                         # per step: each beam's token and its row of the step before
        ended = [[] for _ in prompts]     # (score, ids)
        done = [False] * G
        over = torch.zeros(G, 1, dtype=torch.bool, device=dev)

        def ids_to(step, row):
            out = []
            while step >= 0:
                out.append(int(back[step][0][row]))
                row = int(back[step][1][row])
                step -= 1
            return out[::-1]

        for t in range(int(max_tokens)):
            lg = logits_fn(t, tokens, pages)
            if tuple(lg.shape) != (G * (1 if t == 0 else W), self.vocab):
                raise VsmpError("logits_fn must return [rows, V] logits")
            sel = ctx.beam_select(lg, scores, W, stop_ids=stops)
            token, parent, score, end_token, end_parent, end_score, n_end = (x.cpu().numpy() for x in sel)
            back.append((token.reshape(-1), parent.reshape(-1)))
            length = float(t + 1) ** length_penalty
            for g in range(G):
                if done[g]:
                    continue
                for i in range(int(n_end[g])):
                    ended[g].append((float(end_score[g, i]) / length, ids_to(t - 1, int(end_parent[g, i]))))
                ended[g].sort(key=lambda e: -e[0])
                del ended[g][W:]
                live = token[g, 0] >= 0
                done[g] = not live or (len(ended[g]) == W and ended[g][-1][0] >= float(score[g, 0]) / length)
                if not done[g] and t + 1 == max_tokens:
                    last = [(float(score[g, i]) / length, ids_to(t, g * W + i)) for i in range(W) if token[g, i] >= 0]
                    ended[g] = sorted(ended[g] + last, key=lambda e: -e[0])[:W]
                    done[g] = True
            if all(done):
                break
            over = torch.tensor(done, device=dev).view(G, 1)
            scores = torch.where(over, -float("inf"), sel.score)
            tokens = torch.where(over, -1, sel.token).view(-1)
            rows = sel.parent.view(-1)
            if states is not None:
                ctx.reorder_rows(states, rows * W if t == 0 else rows, W, lens=held)
                if held is not None:
                    held = held + 1
            if pages is not None:  # a beam that is not live, and all of a search that is over, give up their pages
                go = tokens >= 0
                pages, ok = ctx.pages_step(pages, torch.where(go, rows, -1), go.to(torch.int32), cache=cache)
                self.pages = pages
                if not bool(ok.all()):
                    raise VsmpError("the pool has no page left for a beam")
        if pages is not None:
            n = pages.lens.numel()
            self.pages, _ = ctx.pages_step(pages, torch.full((n,), -1, dtype=torch.int32, device=dev))
        return [[(ids, sc) for sc, ids in e] for e in ended]
