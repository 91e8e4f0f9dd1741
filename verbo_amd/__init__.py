"""verbo's token sampler on AMD Instinct MI355X: Python bindings of libvsmp.so (include/vsmp.h).

Mirrors the reference's ctypes layer (python/verbo/__init__.py): a library loader that honours
an environment override, a parameter struct laid out like verbo::Sampling, errors raised from
the library's per-thread message. Device buffers are torch tensors on a ROCm device; only their
addresses cross the C ABI.

    ctx = Context()
    ids = ctx.pick_batch(logits, Params(temp=.8, top_k=50), u_mode=U_COUNTER)  # logits: cuda [B,V]
    s = Sampler(temp=.7, seed=42); s.accept(3); tok = s.pick(numpy_row)        # verbo::Sampler

The operators around the pick (include/vsmp_logits.h):

    x = ctx.head_logits_q4(hidden, q, scales, group)                # 4-bit head: cuda [B, D] -> [B, V]
    x = ctx.adjust_logits(x, Penalty(presence=.5), hist=h, hist_off=o, mask=m, out=x, left=left)
    ids = ctx.pick_batch(x, Params(temp=.8, top_k=50))
    logprob, rank, lse = ctx.logprobs(x, ids[:, None])

Beams and the states behind them (include/vsmp_beam.h):

    step = ctx.beam_select(logits, scores, n, stop_ids=(2,))        # logits: cuda [G * W, V], scores: cuda [G, W]
    ctx.reorder_rows(Planes(caches, token_dim=2), step.parent, n)   # caches: cuda [rows, heads, tokens, width] each
    pages, ok = ctx.pages_step(pages, step.parent, add=1, cache=Planes(pools, token_dim=1))
    pages, moved, live = ctx.pages_compact(pages, cache=Planes(pools, token_dim=1))
"""
import ctypes
import os
from collections import namedtuple
from pathlib import Path

import numpy as np

from .workloads import SAMPLING_DTYPE

__all__ = ["Context", "Sampler", "Params", "Penalty", "PENALTY_DTYPE", "BeamStep", "Planes", "Pages", "RowInfo", "Debug", "VsmpError", "pick_batch_noalloc", "load_library", "U_SUPPLIED", "U_COUNTER",
           "U_XORSHIFT", "ROW_INFO_DTYPE", "SAMPLING_DTYPE"]
__version__ = "0.1.0"

U_SUPPLIED, U_COUNTER, U_XORSHIFT = 0, 1, 2
FLAG_TOPP_NEAR, FLAG_MINP_NEAR, FLAG_DRAW_NEAR, FLAG_FALLBACK = 1, 2, 4, 8
FLAG_SEQ_CUTS, FLAG_CUTS_DIFFER = 16, 32
FLAG_ONE_PASS, FLAG_MINP_PREFIX = 64, 128
PATH_GREEDY, PATH_SMALLK, PATH_GENERAL = 0, 1, 2


class VsmpError(RuntimeError):
    pass


class Params(ctypes.Structure):
    """vsmp_params == verbo::Sampling (reference include/verbo/verbo.hpp:56-64); defaults are the
    reference's."""

    _fields_ = [
        ("temp", ctypes.c_float),
        ("top_k", ctypes.c_int),
        ("top_p", ctypes.c_float),
        ("min_p", ctypes.c_float),
        ("repeat", ctypes.c_float),
        ("repeat_last", ctypes.c_int),
        ("seed", ctypes.c_ulonglong),
    ]

    def __init__(self, temp=0.7, top_k=40, top_p=0.9, min_p=0.0, repeat=1.0, repeat_last=64, seed=0):
        super().__init__(temp, top_k, top_p, min_p, repeat, repeat_last, seed)


class Penalty(ctypes.Structure):
    """vsmp_penalty: what Context.adjust_logits takes from the logits of ids seen before (off by default)."""

    _fields_ = [("repeat", ctypes.c_float), ("presence", ctypes.c_float), ("frequency", ctypes.c_float),
                ("window", ctypes.c_int)]

    def __init__(self, repeat=1.0, presence=0.0, frequency=0.0, window=0):
        super().__init__(repeat, presence, frequency, window)


class RowInfo(ctypes.Structure):
    _fields_ = [
        ("id", ctypes.c_int),
        ("path", ctypes.c_int),
        ("k", ctypes.c_int),
        ("keep_minp", ctypes.c_int),
        ("keep", ctypes.c_int),
        ("rank", ctypes.c_int),
        ("last_id", ctypes.c_int),
        ("flags", ctypes.c_int),
        ("mx", ctypes.c_float),
        ("n_pen", ctypes.c_int),
        ("sum", ctypes.c_double),
        ("tot", ctypes.c_double),
        ("u", ctypes.c_double),
        ("draw_margin", ctypes.c_double),
    ]


class Debug(ctypes.Structure):
    """vsmp_debug: optional diagnostic outputs of vsmp_pick_batch (device addresses)."""

    _fields_ = [
        ("info", ctypes.c_void_p),
        ("cand_ids", ctypes.c_void_p),
        ("cand_pr", ctypes.c_void_p),
        ("cand_cap", ctypes.c_int),
        ("pen_bits", ctypes.c_void_p),
    ]


class _PlanesArg(ctypes.Structure):
    """vsmp_planes."""

    _fields_ = [("planes", ctypes.c_void_p), ("n_planes", ctypes.c_int), ("rows", ctypes.c_int),
                ("row_stride", ctypes.c_longlong), ("pieces", ctypes.c_int), ("piece_stride", ctypes.c_longlong),
                ("tokens", ctypes.c_int), ("token_bytes", ctypes.c_int)]


class _PagesArg(ctypes.Structure):
    """vsmp_pages."""

    _fields_ = [("rows", ctypes.c_int), ("row_pages", ctypes.c_int), ("n_pages", ctypes.c_int),
                ("page_tokens", ctypes.c_int), ("table", ctypes.c_void_p), ("ldt", ctypes.c_longlong),
                ("lens", ctypes.c_void_p), ("ref", ctypes.c_void_p)]


ROW_INFO_DTYPE = np.dtype([("id", "i4"), ("path", "i4"), ("k", "i4"), ("keep_minp", "i4"), ("keep", "i4"),
                           ("rank", "i4"), ("last_id", "i4"), ("flags", "i4"), ("mx", "f4"), ("n_pen", "i4"),
                           ("sum", "f8"), ("tot", "f8"), ("u", "f8"), ("draw_margin", "f8")])
assert ROW_INFO_DTYPE.itemsize == ctypes.sizeof(RowInfo) == 72
assert SAMPLING_DTYPE.itemsize == ctypes.sizeof(Params) == 32
PENALTY_DTYPE = np.dtype([("repeat", "f4"), ("presence", "f4"), ("frequency", "f4"), ("window", "i4")])
assert PENALTY_DTYPE.itemsize == ctypes.sizeof(Penalty) == 16

_lib = None
_P = ctypes.c_void_p


def _candidates():
    env = os.environ.get("VSMP_LIB")
    if env:
        yield Path(env)
    yield Path(__file__).resolve().parent / "libvsmp.so"


def load_library():
    """Load libvsmp.so (VSMP_LIB overrides the in-tree path). Raises VsmpError if it is missing:
    there is no fallback implementation."""
    global _lib
    if _lib is not None:
        return _lib
    # torch ships its own HIP runtime under the same soname (libamdhip64.so.7). Whichever loads
    # first serves the whole process, and torch cannot use a newer one; so when torch is present
    # it is loaded first and this library, its kernels and torch's streams share its runtime.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    for p in _candidates():
        if p.is_file():
            lib = ctypes.CDLL(str(p))
            break
    else:
        raise VsmpError("libvsmp.so not found; build it with `python -m verbo_amd.build` or set VSMP_LIB")
    sig = {
        "vsmp_last_error": (ctypes.c_char_p, []),
        "vsmp_version": (ctypes.c_char_p, []),
        "vsmp_ctx_new": (_P, [ctypes.c_int]),
        "vsmp_ctx_free": (None, [_P]),
        "vsmp_pick_batch": (ctypes.c_int, [_P, _P, ctypes.c_int, ctypes.c_int, ctypes.c_longlong, _P, ctypes.c_int,
                                           _P, _P, ctypes.c_int, _P, _P, ctypes.c_ulonglong, _P,
                                           ctypes.POINTER(Debug), _P]),
        "vsmp_pick_batch_noalloc": (ctypes.c_int, [_P, ctypes.c_int, ctypes.c_int, ctypes.c_longlong, _P, ctypes.c_int,
                                                   _P, _P, ctypes.c_int, _P, _P, ctypes.c_ulonglong, _P,
                                                   ctypes.POINTER(Debug), _P]),
        "vsmp_pick_host": (ctypes.c_int, [_P, _P, ctypes.c_int, ctypes.POINTER(Params), _P, ctypes.c_int,
                                          ctypes.c_double, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(RowInfo)]),
        "vsmp_sampler_new": (_P, [ctypes.POINTER(Params)]),
        "vsmp_sampler_free": (None, [_P]),
        "vsmp_sampler_pick": (ctypes.c_int, [_P, _P, ctypes.c_int]),
        "vsmp_sampler_accept": (None, [_P, ctypes.c_int]),
        "vsmp_sampler_reset": (None, [_P]),
        "vsmp_read_probe": (ctypes.c_int, [_P, _P, ctypes.c_longlong, _P]),
        "vsmp_exp_probe": (ctypes.c_int, [_P, _P, _P, ctypes.c_longlong, _P]),
        "vsmp_numer_probe": (ctypes.c_int, [_P, _P, _P, ctypes.c_longlong, ctypes.c_float, ctypes.c_float, ctypes.c_int,
                                            _P]),
        "vsmp_head_logits": (ctypes.c_int, [_P, _P, ctypes.c_longlong, _P, ctypes.c_longlong, ctypes.c_int, ctypes.c_int,
                                            ctypes.c_int, _P, ctypes.c_longlong, _P]),
        "vsmp_head_pick": (ctypes.c_int, [_P, _P, ctypes.c_longlong, _P, ctypes.c_longlong, ctypes.c_int, ctypes.c_int,
                                          ctypes.c_int, _P, ctypes.c_int, _P, _P, ctypes.c_int, _P, _P,
                                          ctypes.c_ulonglong, _P, _P, ctypes.c_longlong, ctypes.POINTER(Debug), _P]),
        "vsmp_adjust_logits": (ctypes.c_int, [_P, _P, ctypes.c_int, ctypes.c_longlong, ctypes.c_int, ctypes.c_int, _P,
                                              ctypes.c_int, _P, _P, _P, _P, _P, _P, _P, ctypes.c_longlong, ctypes.c_int,
                                              _P, _P, ctypes.c_longlong, _P, _P]),
        "vsmp_logprobs": (ctypes.c_int, [_P, _P, ctypes.c_int, ctypes.c_longlong, ctypes.c_int, ctypes.c_int, _P,
                                         ctypes.c_longlong, ctypes.c_int, _P, _P, _P, _P]),
        "vsmp_head_logits_q4": (ctypes.c_int, [_P, _P, ctypes.c_int, ctypes.c_longlong, _P, ctypes.c_longlong, _P,
                                               ctypes.c_int, ctypes.c_longlong, _P, ctypes.c_longlong, ctypes.c_int,
                                               ctypes.c_int, ctypes.c_int, ctypes.c_int, _P, ctypes.c_longlong, _P]),
        "vsmp_beam_select": (ctypes.c_int, [_P, _P, ctypes.c_int, ctypes.c_longlong, ctypes.c_int, ctypes.c_int,
                                            ctypes.c_int, _P, ctypes.c_int, _P, ctypes.c_int, _P, _P, _P, _P, _P, _P,
                                            _P, _P]),
        "vsmp_reorder_rows": (ctypes.c_int, [_P, _P, _P, ctypes.c_int, _P, _P]),
        "vsmp_pages_step": (ctypes.c_int, [_P, _P, _P, _P, _P, ctypes.c_int, _P, _P, _P]),
        "vsmp_pages_compact": (ctypes.c_int, [_P, _P, _P, _P, _P, _P, _P]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def _err():
    return VsmpError(_lib.vsmp_last_error().decode("utf-8", "replace"))


def version():
    return load_library().vsmp_version().decode()


def _addr(t):
    """Device address of a torch tensor (None stays None)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise VsmpError("expected a device tensor")
    if not t.is_contiguous():
        raise VsmpError("expected a contiguous tensor")
    return t.data_ptr()


DEFAULTS = {"temp": 0.7, "top_k": 40, "top_p": 0.9, "min_p": 0.0, "repeat": 1.0, "repeat_last": 64, "seed": 0}


def params_array(rows=None, n=None, **fields):
    """A SAMPLING_DTYPE array: from a list of dicts/Params, or `n` copies of the given fields
    (missing fields take the reference's defaults)."""
    if rows is None:
        rows = [fields] * int(n or 1)
    out = np.zeros(len(rows), dtype=SAMPLING_DTYPE)
    for i, r in enumerate(rows):
        if isinstance(r, Params):
            r = {f: getattr(r, f) for f, _ in Params._fields_}
        d = dict(DEFAULTS, **r)
        for f in SAMPLING_DTYPE.names:
            out[f][i] = d[f]
    return out


def to_device_params(arr, device="cuda"):
    """Upload a SAMPLING_DTYPE array as a device byte tensor for per-row parameters."""
    import torch

    a = np.ascontiguousarray(arr, dtype=SAMPLING_DTYPE)
    return torch.from_numpy(a.view(np.uint8).copy()).to(device)


def row_info(t):
    """Host numpy ROW_INFO_DTYPE view of a device info tensor (uint8, B*72 bytes)."""
    return t.cpu().numpy().view(ROW_INFO_DTYPE)


def pen_ids(bits, V):
    """Ascending penalised ids per row from a pen_bits bitmap (numpy int32 [B, ceil(V/32)])."""
    b = np.ascontiguousarray(bits).view(np.uint32)
    flat = np.unpackbits(b.view(np.uint8).reshape(b.shape[0], -1), axis=1, bitorder="little")[:, :V]
    return [np.nonzero(r)[0].astype(np.int32) for r in flat]


def _batch_args(logits, params, hist, hist_off, u_mode, u, rng_state, counter, out, info, cand_ids, cand_pr, pen_bits,
                stream):
    """The arguments of vsmp_pick_batch after the context, the output tensor, and the objects whose
    addresses the arguments hold (kept alive by the caller until the call returns)."""
    import torch

    if logits.dim() != 2 or logits.dtype != torch.float32:
        raise VsmpError("logits must be a 2-D float32 device tensor")
    if not logits.is_cuda:
        raise VsmpError("logits must be a device tensor")
    B, V = logits.shape
    ld = logits.stride(0)
    if logits.stride(1) != 1:
        raise VsmpError("logits rows must be contiguous")
    if out is None:
        out = _t().output((B,), torch.int32, logits.device, stream)
    if isinstance(params, Params):
        pp, per_row = ctypes.addressof(params), 0
    else:
        if params.numel() != 32 * B:
            raise VsmpError("per-row params must hold B entries")
        pp, per_row = _addr(params), 1
    cap = cand_ids.shape[1] if cand_ids is not None else 0
    if pen_bits is not None and pen_bits.numel() != B * ((V + 31) // 32):
        raise VsmpError("pen_bits must hold B * ceil(V / 32) words")
    dbg = None
    if info is not None or cand_ids is not None or pen_bits is not None:
        dbg = Debug(_addr(info), _addr(cand_ids), _addr(cand_pr), cap, _addr(pen_bits))
    st = stream if stream is not None else torch.cuda.current_stream(logits.device)
    args = (logits.data_ptr(), B, V, ld, pp, per_row, _addr(hist), _addr(hist_off), int(u_mode), _addr(u),
            _addr(rng_state), int(counter), _addr(out), ctypes.byref(dbg) if dbg is not None else None,
            ctypes.c_void_p(st.cuda_stream))
    return args, out, (params, dbg)


def pick_batch_noalloc(logits, params, hist=None, hist_off=None, u_mode=U_COUNTER, u=None, rng_state=None, counter=0,
                       out=None, info=None, cand_ids=None, cand_pr=None, pen_bits=None, stream=None):
    """vsmp_pick_batch_noalloc: Context.pick_batch's call without a context and without allocating
    (row mode; B <= 2048, V <= 262144; the scratch is a static device array shared by every call on
    the GPU, so calls must not overlap)."""
    load_library()
    args, out, keep = _batch_args(logits, params, hist, hist_off, u_mode, u, rng_state, counter, out, info, cand_ids,
                                  cand_pr, pen_bits, stream)
    if _lib.vsmp_pick_batch_noalloc(*args) != 0:
        raise _err()
    del keep
    return out


def _check_rows(t, dtype, name):
    if not t.is_cuda or t.dtype != dtype or t.dim() != 2 or t.stride(1) != 1:
        raise VsmpError(f"{name} must be a 2-D {dtype} device tensor with contiguous rows")


def _head_shapes(hidden, head):
    """(B, D, V) of a head call on bf16 device tensors hidden [B, D] and head [V, D]."""
    import torch

    _check_rows(hidden, torch.bfloat16, "hidden")
    _check_rows(head, torch.bfloat16, "head")
    if hidden.shape[1] != head.shape[1]:
        raise VsmpError("hidden and head must have the same number of columns (D)")
    return hidden.shape[0], hidden.shape[1], head.shape[0]


class _Torch:
    """What the calls below need of torch, looked up once: they are short enough for an import statement and a
    Stream object per call to show."""

    def __init__(self):
        import torch

        self.empty, self.int32, self.float32, self.uint8 = torch.empty, torch.int32, torch.float32, torch.uint8
        self.codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # vsmp_dtype
        self._raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._current = torch.cuda.current_stream
        self._use, self._external, self._default = torch.cuda.stream, torch.cuda.ExternalStream, torch.cuda.default_stream

    def stream(self, stream, device):
        """The address of `stream`, or of torch's current one on `device`."""
        if stream is not None:
            return stream.cuda_stream
        return self._raw(device.index) if self._raw is not None else self._current(device).cuda_stream

    def _at(self, address, device):
        """The stream at an address: of a stream, the calls ask for no more than that. (Made from the default stream's,
        0, an ExternalStream would be a new one.)"""
        return self._external(address, device=device) if address else self._default(device)

    def output(self, shape, dtype, device, stream):
        """A new tensor that a call on `stream` (None: the current one) writes. On a stream of its own the call takes
        that stream's memory, since the current one may still be using what it has freed; once the tensor is freed,
        the memory waits for the work of both."""
        if stream is None or stream.cuda_stream == self.stream(None, device):
            return self.empty(shape, dtype=dtype, device=device)
        with self._use(self._at(stream.cuda_stream, device)):
            t = self.empty(shape, dtype=dtype, device=device)
        t.record_stream(self._current(device))
        return t

    def rows16(self, B, V, device, stream):
        """Such an output of float32 [B, V] whose rows are padded to 16 bytes, and their stride."""
        ld = (V + 3) // 4 * 4
        t = self.output((B, ld), self.float32, device, stream)
        return (t if ld == V else t[:, :V]), ld


_torch = None


def _t():
    global _torch
    if _torch is None:
        _torch = _Torch()
    return _torch


def _rows_of(t, name, device):
    """(dtype code, row stride) of a 2-D matrix with contiguous rows on `device` (of a single row: its length)."""
    code = _t().codes.get(t.dtype)
    if code is None:
        raise VsmpError(f"{name} must be float32, bfloat16 or float16")
    if t.dim() != 2 or not t.is_cuda or t.device != device:
        raise VsmpError(f"{name} must be a 2-D tensor on {device}")
    rows, cols = t.shape
    sr, sc = t.stride()
    if cols > 1 and sc != 1:
        raise VsmpError(f"{name} must have contiguous rows")
    return code, sr if rows > 1 else cols


def _array_of(t, dtype, n, name, device):
    """The address of a contiguous device array of `dtype` with at least n entries (None stays None)."""
    if t is None:
        return None
    if t.dtype != dtype or t.device != device or not t.is_contiguous() or t.numel() < n:
        raise VsmpError(f"{name} must be a contiguous {dtype} tensor on {device} of at least {n} entries")
    return t.data_ptr()


def _int32(v, name):
    """v as an int that a C int holds (ctypes would cut it)."""
    v = int(v)
    if not -1 << 31 <= v < 1 << 31:
        raise VsmpError(f"{name} must fit 32 bits")
    return v


def _penalty_rows(rows):
    """A PENALTY_DTYPE array of such an array or of a list of Penalty, each of them what a shared one has to be."""
    if not isinstance(rows, np.ndarray):
        rows = np.array([(p.repeat, p.presence, p.frequency, p.window) for p in rows], dtype=PENALTY_DTYPE)
    a = np.ascontiguousarray(rows, dtype=PENALTY_DTYPE)
    if not all(np.isfinite(a[f]).all() for f in ("repeat", "presence", "frequency")) or not (a["repeat"] > 0).all():
        raise VsmpError("penalties must be finite, repeat above 0")
    return a


def to_device_penalties(rows, device="cuda"):
    """Upload a PENALTY_DTYPE array, or a list of Penalty (finite, repeat above 0), as a device byte tensor for per-row
    penalties."""
    import torch

    return torch.from_numpy(_penalty_rows(rows).view(np.uint8).copy()).to(device)


def _adjust_args(logits, penalty, hist, hist_off, prompt_len, bias_ids, bias, bias_off, mask, mask_row, out, left, stream,
                 csr=True):
    """The arguments of an adjust call as (in, dtype, ldi), (B, V), the penalties, histories, and the rest up to the
    stream; `out`; and what the addresses need kept alive."""
    T = _t()
    dev = logits.device
    code, ld = _rows_of(logits, "logits", dev)
    B, V = logits.shape
    if out is None:  # rows on 16 bytes, so that pick_batch can take them
        out, ldo = T.rows16(B, V, dev, stream)
    else:
        ocode, ldo = _rows_of(out, "out", dev)
        if ocode != 0 or out.shape != logits.shape:
            raise VsmpError("out must be float32 of the logits' shape")
    i32 = T.int32
    if penalty is None or isinstance(penalty, Penalty):
        pp, per_row = (ctypes.addressof(penalty) if penalty is not None else None), 0
    else:
        if penalty.dtype != T.uint8 or penalty.numel() != 16 * B:
            raise VsmpError("per-row penalties must hold B entries (to_device_penalties)")
        pp, per_row = _array_of(penalty, T.uint8, 16 * B, "per-row penalties", dev), 1
    if csr:
        if (hist is None) != (hist_off is None):
            raise VsmpError("hist and hist_off go together")
        if hist is not None and hist.numel() == 0:  # every history is empty
            hist = hist_off = prompt_len = None
        h, ho = _array_of(hist, i32, 0, "hist", dev), _array_of(hist_off, i32, B + 1, "hist_off", dev)
    else:
        h = ho = None
    if (bias_ids is None) != (bias_off is None) or (bias is None) != (bias_off is None):
        raise VsmpError("bias_ids, bias and bias_off go together")
    if bias_ids is not None and bias_ids.numel() == 0:
        bias_ids = bias = bias_off = None
    ldm = n_masks = 0
    mp = None
    if mask is not None:
        if mask.dtype != i32 or mask.dim() != 2 or mask.device != dev or mask.stride(1) != 1 or mask.shape[1] < (V + 31) // 32:
            raise VsmpError("mask must be an int32 tensor [masks, >= ceil(V / 32)] with contiguous rows on the logits' device")
        n_masks = mask.shape[0]
        if n_masks < 1:  # its address would be NULL, which is no masks at all
            raise VsmpError("mask must hold at least one mask")
        ldm = mask.stride(0) if n_masks > 1 else mask.shape[1]
        mp = mask.data_ptr()
    rest = (_array_of(prompt_len, i32, B, "prompt_len", dev), _array_of(bias_ids, i32, 0, "bias_ids", dev),
            _array_of(bias, T.float32, bias_ids.numel() if bias_ids is not None else 0, "bias", dev),
            _array_of(bias_off, i32, B + 1, "bias_off", dev), mp, ldm, n_masks,
            _array_of(mask_row, i32, B, "mask_row", dev), out.data_ptr(), ldo, _array_of(left, i32, B, "left", dev),
            T.stream(stream, dev))
    return (logits.data_ptr(), code, ld), (B, V), (pp, per_row), (h, ho), rest, out


_Stops = ctypes.c_int * 16  # the most stop tokens of a selection
BeamStep = namedtuple("BeamStep", "token parent score end_token end_parent end_score n_end")
BeamStep.__doc__ = """What Context.beam_select returns: for each group the n best continuations that go on (token, parent: the
row, both int32 [G, n]; score: float32 [G, n]) and those that a stop token ends (the same, n_end of them: int32 [G])."""


class Planes:
    """vsmp_planes: device tensors of one shape, strides and type whose rows (dimension 0) hold tokens, such as the keys
    and values of every layer. Making them uploads the tensors' addresses and waits for the current stream, so that a program
    keeps them as long as the tensors, and as long as it replays graphs of calls with them. token_dim: the dimension that counts tokens, with a
    token's values side by side behind it and whole tokens one after the other; None: a row is one token, whole.
    Dimensions before it must have one stride in common (heads that lie apart)."""

    def __init__(self, tensors, token_dim=None):
        import torch

        self.tensors = list(tensors)
        if not self.tensors:
            raise VsmpError("planes need at least one tensor")
        t = self.tensors[0]
        if not t.is_cuda or t.dim() < 1 or t.numel() == 0:
            raise VsmpError("planes must be device tensors with at least one row and element")
        for u in self.tensors:
            if u.shape != t.shape or u.stride() != t.stride() or u.dtype != t.dtype or u.device != t.device:
                raise VsmpError("planes must have one shape, one type, the same strides and one device")
        if len(set(u.data_ptr() for u in self.tensors)) != len(self.tensors):
            raise VsmpError("planes must be tensors of their own")
        size, n = t.element_size(), t.dim()
        dim = None if token_dim is None else int(token_dim) + (n if token_dim < 0 else 0)
        if dim is not None and not 1 <= dim < n:
            raise VsmpError("token_dim must be a dimension of the planes behind the first")

        def together(dims):
            """(entries, stride) of dimensions that one stride walks through; None if none does."""
            dims = [(k, d) for k, d in dims if k > 1]
            if any(a[1] != b[0] * b[1] for a, b in zip(dims, dims[1:])):
                return None
            count = 1
            for k, _ in dims:
                count *= k
            return count, dims[-1][1] if dims else 0

        shape, stride = t.shape, t.stride()
        dims = list(zip(shape, stride))
        cut = dim + 1 if dim is not None else n
        if dim is None:  # as many of the last dimensions as lie side by side
            width = 1
            while cut > 1 and (shape[cut - 1] == 1 or stride[cut - 1] == width):
                cut -= 1
                width *= shape[cut]
            tokens, token = 1, width
            inner, outer = (width, 1), together(dims[1:cut])
        else:
            inner = together(dims[cut:])
            tokens, token = shape[dim], inner[0] if inner else 0
            outer = together(dims[1:dim])
        if inner is None or (inner[0] > 1 and inner[1] != 1) or (tokens > 1 and stride[dim] != token):
            raise VsmpError("a token's values must lie side by side, and tokens one after the other")
        if outer is None:
            raise VsmpError("the dimensions before the tokens must have one stride in common")
        for v, name in ((shape[0], "rows"), (outer[0], "pieces"), (tokens, "tokens"), (token * size, "a token's bytes")):
            _int32(v, name)
        self.device, self.rows, self.tokens, self.token_dim = t.device, shape[0], tokens, dim
        self._ptrs = torch.tensor([u.data_ptr() for u in self.tensors], dtype=torch.int64).to(t.device)
        # the addresses are there for every stream from here on
        torch.cuda.current_stream(t.device).synchronize()
        self._streams = {_t().stream(None, t.device)}
        self._arg = _PlanesArg(self._ptrs.data_ptr(), len(self.tensors), shape[0], stride[0] * size if shape[0] > 1 else 0, outer[0],
                               outer[1] * size, tokens, token * size)
        self._addr = ctypes.addressof(self._arg)

    def _on(self, address):
        """The planes for a call on the stream at that address: where that is not the one they were made on, the addresses'
        memory waits for it too when the planes are gone."""
        if address not in self._streams:
            self._ptrs.record_stream(_t()._at(address, self.device))
            self._streams.add(address)
        return self._addr


class Pages:
    """vsmp_pages: a cache in pages as its rows use it. table: int32 [rows, row_pages], a row's page numbers (contiguous
    rows); lens: int32 [rows], its tokens; ref: int32 [n_pages], how many hold each page; page_tokens: tokens of a page.
    The tensors are the program's; Context.pages_step and pages_compact read one such state and write another."""

    def __init__(self, table, lens, ref, page_tokens):
        T = _t()
        dev = table.device
        if table.dtype != T.int32 or table.dim() != 2 or not table.is_cuda or (table.shape[1] > 1 and table.stride(1) != 1):
            raise VsmpError("table must be a 2-D int32 device tensor with contiguous rows")
        rows, cap = table.shape
        for t, name in ((lens, "lens"), (ref, "ref")):
            if t.dim() != 1:
                raise VsmpError(f"{name} must be one-dimensional")
            _array_of(t, T.int32, rows if name == "lens" else 1, name, dev)
        if lens.numel() != rows:
            raise VsmpError("lens must hold an entry for each row of the table")
        self.table, self.lens, self.ref, self.page_tokens, self.device = table, lens, ref, _int32(page_tokens, "page_tokens"), dev
        self._arg = _PagesArg(_int32(rows, "rows"), _int32(cap, "row_pages"), _int32(ref.numel(), "n_pages"), self.page_tokens,
                              table.data_ptr(), table.stride(0) if rows > 1 else cap, lens.data_ptr(), ref.data_ptr())
        self._addr = ctypes.addressof(self._arg)

    @classmethod
    def empty(cls, rows, row_pages, n_pages, page_tokens, device="cuda"):
        """A pool of free pages, and rows without tokens."""
        import torch

        return cls(torch.full((rows, row_pages), -1, dtype=torch.int32, device=device), torch.zeros(rows, dtype=torch.int32, device=device),
                   torch.zeros(n_pages, dtype=torch.int32, device=device), page_tokens)

    def like(self, rows=None, stream=None):
        """Memory for a state of this pool, of as many rows or of `rows`: what a step writes into. `stream`: that of the
        step."""
        T = _t()
        n = self.lens.numel() if rows is None else int(rows)
        return Pages(T.output((n, self.table.shape[1]), T.int32, self.device, stream), T.output((n,), T.int32, self.device, stream),
                     T.output((self.ref.numel(),), T.int32, self.device, stream), self.page_tokens)


class Context:
    """A vsmp_ctx on one device: scratch for batched picks, staging for host picks."""

    def __init__(self, device=0):
        load_library()
        self._h = _lib.vsmp_ctx_new(int(device))
        if not self._h:
            raise _err()
        self.device = device

    def close(self):
        h = getattr(self, "_h", None)
        if h and _lib is not None:
            _lib.vsmp_ctx_free(h)
            self._h = None

    def __del__(self):
        self.close()

    def pick_batch(self, logits, params, hist=None, hist_off=None, u_mode=U_COUNTER, u=None, rng_state=None,
                   counter=0, out=None, info=None, cand_ids=None, cand_pr=None, pen_bits=None, stream=None):
        """vsmp_pick_batch on torch device tensors. `params`: a Params (shared by all rows) or a
        device byte tensor from to_device_params (one entry per row). Returns `out` (int32 [B]).
        Diagnostics (vsmp_debug): info (uint8 [B*72]), cand_ids (int32 [B, cap]) / cand_pr (float64
        [B, cap]), pen_bits (int32 [B, ceil(V/32)]).
        Stream-ordered on `stream` (default: torch's current stream); does not synchronise."""
        args, out, keep = _batch_args(logits, params, hist, hist_off, u_mode, u, rng_state, counter, out, info,
                                      cand_ids, cand_pr, pen_bits, stream)
        if _lib.vsmp_pick_batch(self._h, *args) != 0:
            raise _err()
        del keep
        return out

    def head_logits(self, hidden, head, logits=None, stream=None):
        """vsmp_head_logits: logits = hidden @ head.T for bf16 device tensors hidden [B, D] and head
        [V, D] (rows contiguous), fp32 accumulation; returns logits (float32 [B, V] unless given)."""
        import torch

        B, D, V = _head_shapes(hidden, head)
        if logits is None:  # rows padded to 16 bytes, so that pick_batch can take them
            logits = _t().rows16(B, V, hidden.device, stream)[0]
        _check_rows(logits, torch.float32, "logits")
        st = stream if stream is not None else torch.cuda.current_stream(hidden.device)
        if _lib.vsmp_head_logits(self._h, hidden.data_ptr(), hidden.stride(0), head.data_ptr(), head.stride(0), B, V, D,
                                 logits.data_ptr(), logits.stride(0), ctypes.c_void_p(st.cuda_stream)) != 0:
            raise _err()
        return logits

    def head_pick(self, hidden, head, params, hist=None, hist_off=None, u_mode=U_COUNTER, u=None, rng_state=None,
                  counter=0, out=None, logits=None, info=None, cand_ids=None, cand_pr=None, pen_bits=None, stream=None):
        """vsmp_head_pick: the head's product and pick_batch's pick in one call (the ids pick_batch
        takes from head_logits' logits). `logits`: None, or a float32 [B, >= V] device tensor that
        receives the logits as well. The rest as pick_batch. Returns `out` (int32 [B])."""
        import torch

        B, D, V = _head_shapes(hidden, head)
        if out is None:
            out = _t().output((B,), torch.int32, hidden.device, stream)
        if logits is not None:
            _check_rows(logits, torch.float32, "logits")
        if isinstance(params, Params):
            pp, per_row = ctypes.addressof(params), 0
        else:
            if params.numel() != 32 * B:
                raise VsmpError("per-row params must hold B entries")
            pp, per_row = _addr(params), 1
        cap = cand_ids.shape[1] if cand_ids is not None else 0
        if pen_bits is not None and pen_bits.numel() != B * ((V + 31) // 32):
            raise VsmpError("pen_bits must hold B * ceil(V / 32) words")
        dbg = None
        if info is not None or cand_ids is not None or pen_bits is not None:
            dbg = Debug(_addr(info), _addr(cand_ids), _addr(cand_pr), cap, _addr(pen_bits))
        st = stream if stream is not None else torch.cuda.current_stream(hidden.device)
        rc = _lib.vsmp_head_pick(self._h, hidden.data_ptr(), hidden.stride(0), head.data_ptr(), head.stride(0), B, V, D,
                                 pp, per_row, _addr(hist), _addr(hist_off), int(u_mode), _addr(u), _addr(rng_state),
                                 int(counter), _addr(out), logits.data_ptr() if logits is not None else None,
                                 logits.stride(0) if logits is not None else 0,
                                 ctypes.byref(dbg) if dbg is not None else None, ctypes.c_void_p(st.cuda_stream))
        if rc != 0:
            raise _err()
        del params, dbg
        return out

    def _check_device(self, t):
        if not t.is_cuda or (self.device >= 0 and t.device.index != self.device):
            raise VsmpError(f"expected tensors on the context's device ({self.device})")

    def adjust_logits(self, logits, penalty=None, hist=None, hist_off=None, prompt_len=None, bias_ids=None, bias=None,
                      bias_off=None, mask=None, mask_row=None, out=None, left=None, stream=None):
        """vsmp_adjust_logits: penalties for repeated tokens, biases and grammar masks on device logits [B, V]
        (float32, bfloat16 or float16; rows contiguous). `penalty`: a Penalty (shared by all rows) or a device
        byte tensor from to_device_penalties; hist / hist_off / prompt_len (int32): CSR histories and the length of
        each one's prompt; bias_ids (int32) / bias (float32) / bias_off (int32): CSR biases; mask (int32 [masks,
        ceil(V / 32)], bits set for allowed tokens) and mask_row (int32 [B], negative: none). `out`: None, a float32
        [B, V] tensor, or `logits` itself; `left`: None, or int32 [B] for the number of tokens left in each row.
        Returns `out`, whose rows pick_batch can take."""
        self._check_device(logits)
        x, shape, pen, hists, rest, out = _adjust_args(logits, penalty, hist, hist_off, prompt_len, bias_ids, bias, bias_off,
                                                       mask, mask_row, out, left, stream)
        if _lib.vsmp_adjust_logits(self._h, *x, *shape, *pen, *hists, *rest) != 0:
            raise _err()
        return out

    def logprobs(self, logits, ids=None, rank=True, stream=None):
        """vsmp_logprobs: the log-probabilities of ids (int32 [B, n], n <= 64, rows contiguous) under the softmax of
        device logits [B, V] (float32, bfloat16 or float16), their ranks in the sampler's order (rank=False: None)
        and each row's log of the sum of exponentials. Ids outside [0, V) give -inf and rank -1. Returns (logprob
        float32 [B, n], rank int32 [B, n], lse float32 [B]); without ids the first two are None."""
        T = _t()
        self._check_device(logits)
        dev = logits.device
        code, ld = _rows_of(logits, "logits", dev)
        B, V = logits.shape
        lse = T.output((B,), T.float32, dev, stream)
        lp = rk = None
        n = ldj = 0
        if ids is not None:
            if ids.dtype != T.int32 or ids.dim() != 2 or ids.shape[0] != B or ids.device != dev:
                raise VsmpError("ids must be an int32 tensor [B, n] on the logits' device")
            n = ids.shape[1]
            if n > 1 and ids.stride(1) != 1:
                raise VsmpError("ids must have contiguous rows")
            ldj = ids.stride(0) if B > 1 else n
            lp = T.output((B, n), T.float32, dev, stream)
            rk = T.output((B, n), T.int32, dev, stream) if rank else None
        if _lib.vsmp_logprobs(self._h, logits.data_ptr(), code, ld, B, V, ids.data_ptr() if n else None, ldj, n,
                              lp.data_ptr() if n else None, rk.data_ptr() if n and rk is not None else None,
                              lse.data_ptr(), T.stream(stream, dev)) != 0:
            raise _err()
        return lp, rk, lse

    def head_logits_q4(self, hidden, q, scales, group, zeros=None, logits=None, stream=None):
        """vsmp_head_logits_q4: the head's product with 4-bit weights, logits = hidden @ W.T with W[c, d] =
        scales[c, d / group] * (q[c, d] - zeros[c, d / group]). hidden: bfloat16 or float16 [B, D]; q: uint8
        [V, D / 2], two weights a byte, the even d in the low half; scales: float32, bfloat16 or float16 [V, D /
        group]; zeros: uint8 [V, D / group], or None for 8. Returns logits (float32 [B, V] unless given)."""
        T = _t()
        self._check_device(hidden)
        dev = hidden.device
        code, ldh = _rows_of(hidden, "hidden", dev)
        if code == 0:
            raise VsmpError("hidden must be bfloat16 or float16")
        B, D = hidden.shape
        if q.dtype != T.uint8 or q.dim() != 2 or q.device != dev or (q.shape[1] > 1 and q.stride(1) != 1):
            raise VsmpError("q must be a 2-D uint8 tensor with contiguous rows on the hidden states' device")
        V = q.shape[0]
        if 2 * q.shape[1] != D:
            raise VsmpError("q must hold D / 2 bytes per row")
        scode, lds = _rows_of(scales, "scales", dev)
        group = int(group)
        if group < 1 or scales.shape != (V, D // group):
            raise VsmpError("scales must be [V, D / group]")
        ldz = 0
        if zeros is not None:
            if zeros.dtype != T.uint8 or zeros.shape != scales.shape or zeros.device != dev or \
                    (zeros.shape[1] > 1 and zeros.stride(1) != 1):
                raise VsmpError("zeros must be uint8 of the scales' shape with contiguous rows")
            ldz = zeros.stride(0) if V > 1 else zeros.shape[1]
        if logits is None:  # rows padded to 16 bytes, so that pick_batch can take them
            logits, ldl = T.rows16(B, V, dev, stream)
        else:
            lcode, ldl = _rows_of(logits, "logits", dev)
            if lcode != 0 or logits.shape != (B, V):
                raise VsmpError("logits must be float32 [B, V]")
        if _lib.vsmp_head_logits_q4(self._h, hidden.data_ptr(), code, ldh, q.data_ptr(),
                                    q.stride(0) if V > 1 else D // 2,
                                    scales.data_ptr(), scode, lds, zeros.data_ptr() if zeros is not None else None, ldz,
                                    group, B, V, D, logits.data_ptr(), ldl, T.stream(stream, dev)) != 0:
            raise _err()
        return logits

    def beam_select(self, logits, scores, n=None, stop_ids=(), stream=None):
        """vsmp_beam_select: one step of beam search. logits: device [G * W, V] (float32, bfloat16 or float16; rows
        contiguous), the rows of a group one after the other; scores: float32 [G, W], -inf for a row that is not live;
        n: beams of the next step (default W); stop_ids: at most 16 tokens that end a sequence. Returns a BeamStep."""
        T = _t()
        self._check_device(logits)
        dev = logits.device
        code, ld = _rows_of(logits, "logits", dev)
        B, V = logits.shape
        if scores.dim() != 2 or scores.numel() != B:
            raise VsmpError("scores must be a float32 tensor [G, W] with an entry for each row of logits")
        G, W = scores.shape
        n = W if n is None else int(n)
        if n < 1:
            raise VsmpError("need n >= 1 beams of the next step")
        if (B | V | n) >> 31:
            raise VsmpError("logits' sizes and n must fit 32 bits")
        ns = len(stop_ids)
        # (those outside the vocabulary end nothing, also where a C int would not hold them)
        stops = (_Stops if ns <= 16 else ctypes.c_int * ns)(*[t if 0 <= t < V else -1 for t in stop_ids]) if ns else None
        sp = _array_of(scores, T.float32, B, "scores", dev)
        token, parent, end_token, end_parent, score, end_score = T.output((6, G, n), T.int32, dev, stream).unbind(0)
        n_end = T.output((G,), T.int32, dev, stream)
        p, k = token.data_ptr(), 4 * G * n  # the six lie one after the other
        if _lib.vsmp_beam_select(self._h, logits.data_ptr(), code, ld, G, W, V, sp, n, stops, ns, p, p + k, p + 4 * k, p + 2 * k,
                                 p + 3 * k, p + 5 * k, n_end.data_ptr(), T.stream(stream, dev)) != 0:
            raise _err()
        score, end_score = score.view(T.float32), end_score.view(T.float32)
        return BeamStep(token, parent, score, end_token, end_parent, end_score, n_end)

    def reorder_rows(self, planes, parent, width, lens=None, stream=None):
        """vsmp_reorder_rows: in every plane of `planes` (a Planes) row i takes what row parent[i] held, in place. parent:
        int32 [rows], row numbers within each group of `width` rows; others leave their row as it is. lens: int32
        [rows], the tokens that each row held before; None: all."""
        T = _t()
        dev = planes.device
        if self.device >= 0 and dev.index != self.device:
            raise VsmpError(f"expected tensors on the context's device ({self.device})")
        st = T.stream(stream, dev)
        if _lib.vsmp_reorder_rows(self._h, planes._on(st), _array_of(parent, T.int32, planes.rows, "parent", dev), _int32(width, "width"),
                                  _array_of(lens, T.int32, planes.rows, "lens", dev), st) != 0:
            raise _err()

    def _pages(self, pages, cache, stream):
        dev, st = pages.device, _t().stream(stream, pages.device)
        if self.device >= 0 and dev.index != self.device:
            raise VsmpError(f"expected tensors on the context's device ({self.device})")
        if cache is not None and cache.device != dev:
            raise VsmpError("the cache must be on the pages' device")
        return dev, st, cache._on(st) if cache is not None else None

    def pages_step(self, pages, parent=None, add=0, cache=None, out=None, stream=None):
        """vsmp_pages_step: the step of a cache in pages from the state `pages` (a Pages, left as it is). Row i takes the
        pages of row parent[i] (int32, one for each row of the next state; None: its own; outside the rows: none) and
        grows by add[i] tokens, or is cut by -add[i] (an int32 tensor, or an int for every row). cache: a Planes whose
        rows are the pages, so that begun pages which rows share are copied; None: tables alone. out: a Pages for the
        next state (default: new, a row for each parent). Returns (the next state, ok int32 [rows]: 0 for a row that
        did not get its pages; from the first row on that the pool has too few for, no row gets any in that step)."""
        T = _t()
        dev, st, cp = self._pages(pages, cache, stream)
        if out is None:
            out = pages.like(None if parent is None else parent.numel(), stream)
        rows = out.lens.numel()
        every = 0
        if not hasattr(add, "data_ptr"):
            add, every = None, _int32(add, "add")
        ok = T.output((rows,), T.int32, dev, stream)
        if out.device != dev:
            raise VsmpError("out must be on the pages' device")
        if _lib.vsmp_pages_step(self._h, pages._addr, out._addr, _array_of(parent, T.int32, rows, "parent", dev),
                                _array_of(add, T.int32, rows, "add", dev), every, cp, ok.data_ptr(), st) != 0:
            raise _err()
        return out, ok

    def pages_compact(self, pages, cache=None, out=None, stream=None):
        """vsmp_pages_compact: the pages in use moved together into the pool's first, from the state `pages` (left as it
        is), in every plane of `cache`. Returns (the next state: `out`, or a new Pages; moved int32 [n_pages]: each
        page's new number, -1 for a free one; live int32 [1]: how many are in use)."""
        T = _t()
        dev, st, cp = self._pages(pages, cache, stream)
        if out is None:
            out = pages.like(stream=stream)
        if out.device != dev:
            raise VsmpError("out must be on the pages' device")
        n = pages.ref.numel()
        moved, live = T.output((n,), T.int32, dev, stream), T.output((1,), T.int32, dev, stream)
        if _lib.vsmp_pages_compact(self._h, pages._addr, out._addr, cp, moved.data_ptr(), live.data_ptr(), st) != 0:
            raise _err()
        return out, moved, live

    def read_probe(self, t, stream=None):
        """vsmp_read_probe: stream the bytes of device tensor `t` through a plain read kernel on
        `stream` (default: torch's current stream). For measuring attainable read bandwidth."""
        import torch

        st = stream if stream is not None else torch.cuda.current_stream(t.device)
        nbytes = t.numel() * t.element_size() // 16 * 16
        if _lib.vsmp_read_probe(self._h, t.data_ptr(), nbytes, ctypes.c_void_p(st.cuda_stream)) != 0:
            raise _err()

    def exp_probe(self, x, stream=None):
        """vsmp_exp_probe: the general path's fp64 exp over device tensor `x` (float64); returns y."""
        import torch

        if x.dtype != torch.float64 or not x.is_cuda:
            raise VsmpError("exp_probe needs a float64 device tensor")
        x = x.contiguous()
        y = torch.empty_like(x)
        st = stream if stream is not None else torch.cuda.current_stream(x.device)
        if _lib.vsmp_exp_probe(self._h, x.data_ptr(), y.data_ptr(), x.numel(), ctypes.c_void_p(st.cuda_stream)) != 0:
            raise _err()
        return y

    def numer_probe(self, d, temp, qs, fixed_point=False, stream=None):
        """vsmp_numer_probe: the general path's numerators exp(double(d) / temp) for float32 device
        tensor `d` (= v - max <= 0), buckets of scale qs: the table numerators, or with fixed_point
        each element's share of its bucket's mass; returns float64 y."""
        import torch

        if d.dtype != torch.float32 or not d.is_cuda:
            raise VsmpError("numer_probe needs a float32 device tensor")
        d = d.contiguous()
        y = torch.empty(d.shape, dtype=torch.float64, device=d.device)
        st = stream if stream is not None else torch.cuda.current_stream(d.device)
        if _lib.vsmp_numer_probe(self._h, d.data_ptr(), y.data_ptr(), d.numel(), float(temp), float(qs),
                                 1 if fixed_point else 0, ctypes.c_void_p(st.cuda_stream)) != 0:
            raise _err()
        return y

    def pick_host(self, logits, params, hist=(), u=0.0, with_info=False):
        """vsmp_pick_host: one pick on a host row (numpy). Returns id (and RowInfo)."""
        lg = np.ascontiguousarray(logits, dtype=np.float32)
        h = np.ascontiguousarray(hist, dtype=np.int32)
        out = ctypes.c_int(-1)
        info = RowInfo()
        rc = _lib.vsmp_pick_host(self._h, lg.ctypes.data_as(_P), lg.size, ctypes.byref(params),
                                 h.ctypes.data_as(_P) if h.size else None, h.size, float(u), ctypes.byref(out),
                                 ctypes.byref(info) if with_info else None)
        if rc != 0:
            raise _err()
        return (out.value, info) if with_info else out.value


class Sampler:
    """verbo::Sampler (reference include/verbo/verbo.hpp:116-132) with pick on the GPU."""

    def __init__(self, params=None, **kw):
        load_library()
        p = params if params is not None else Params(**kw)
        self._h = _lib.vsmp_sampler_new(ctypes.byref(p))
        if not self._h:
            raise _err()

    def __del__(self):
        h = getattr(self, "_h", None)
        if h and _lib is not None:
            _lib.vsmp_sampler_free(h)
            self._h = None

    def pick(self, logits):
        lg = np.ascontiguousarray(logits, dtype=np.float32)
        # the address as a plain int: ndarray.ctypes.data_as builds several objects per call
        r = _lib.vsmp_sampler_pick(self._h, lg.ctypes.data, lg.size)
        if r < 0:
            raise _err()
        return r

    def accept(self, tok):
        _lib.vsmp_sampler_accept(self._h, int(tok))

    def reset(self):
        _lib.vsmp_sampler_reset(self._h)
