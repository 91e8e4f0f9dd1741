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
"""
import ctypes
import os
from pathlib import Path

import numpy as np

from .workloads import SAMPLING_DTYPE

__all__ = ["Context", "Sampler", "Params", "Penalty", "PENALTY_DTYPE", "RowInfo", "Debug", "VsmpError", "pick_batch_noalloc", "load_library", "U_SUPPLIED", "U_COUNTER",
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
        self._use, self._external = torch.cuda.stream, torch.cuda.ExternalStream

    def stream(self, stream, device):
        """The address of `stream`, or of torch's current one on `device`."""
        if stream is not None:
            return stream.cuda_stream
        return self._raw(device.index) if self._raw is not None else self._current(device).cuda_stream

    def output(self, shape, dtype, device, stream):
        """A new tensor that a call on `stream` (None: the current one) writes. On a stream of its own the call takes
        that stream's memory, since the current one may still be using what it has freed; once the tensor is freed,
        the memory waits for the work of both."""
        if stream is None or stream.cuda_stream == self.stream(None, device):
            return self.empty(shape, dtype=dtype, device=device)
        # by its address: of a stream, the calls ask for no more than that
        with self._use(self._external(stream.cuda_stream, device=device)):
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
