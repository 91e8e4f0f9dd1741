"""The operators around the pick on the CPU: every declared entry point is exported, the header compiles as C, the
penalty struct has its layout, and bad arguments are refused with a message before any GPU work. No GPU calls."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import verbo_amd as V
from verbo_amd import decode

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "vsmp_logits.h"


def test_entry_points_are_declared_and_exported():
    names = re.findall(r"VSMP_API\s+[\w\s\*]+?\b(vsmp_\w+)\s*\(", HEADER.read_text())
    assert names == ["vsmp_adjust_logits", "vsmp_logprobs", "vsmp_head_logits_q4", "vsmp_bsampler_adjust_rows"]
    lib = V.load_library()
    for n in names:
        assert hasattr(lib, n), n


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc absent")
def test_header_compiles_as_c_and_the_struct_has_its_layout(tmp_path):
    src = tmp_path / "h.c"
    src.write_text("#include <stddef.h>\n#include \"vsmp_logits.h\"\n"
                   "_Static_assert(sizeof(vsmp_penalty) == 16, \"size\");\n"
                   "_Static_assert(offsetof(vsmp_penalty, window) == 12, \"window\");\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"), "-c", str(src), "-o",
                    str(tmp_path / "h.o")], check=True)
    assert ctypes.sizeof(V.Penalty) == V.PENALTY_DTYPE.itemsize == 16
    assert V.Penalty.window.offset == V.PENALTY_DTYPE.fields["window"][1] == 12
    p = V.Penalty()
    assert (p.repeat, p.presence, p.frequency, p.window) == (1.0, 0.0, 0.0, 0)


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ absent")
def test_the_documented_step_compiles(tmp_path):
    """The C++ block that INTEGRATION.md shows for these calls, with the variables that it names."""
    block = [b for b in re.findall(r"```cpp\n(.*?)```", (ROOT / "INTEGRATION.md").read_text(), re.S) if "vsmp_logits.h" in b]
    assert len(block) == 1
    body = "\n".join(line for line in block[0].splitlines() if not line.startswith("#include"))
    src = tmp_path / "step.cpp"
    src.write_text("""#include "vsmp_logits.h"
void step(vsmp_ctx* ctx, const void* d_hidden, long long ldh, const void* d_q, long long ldq, const void* d_scales, int B, int V,
          int D, float* d_logits, long long ld, void* stream, const int* d_hist, const int* d_hist_off, const int* d_prompt_len,
          const int* d_bias_ids, const float* d_bias, const int* d_bias_off, const unsigned* d_mask, long long ldm, int n_masks,
          const int* d_mask_row, int* d_left, vsmp_params params, unsigned long long step, int* d_ids, float* d_logprob,
          int* d_rank, float* d_lse) {
""" + body + "\n}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"), "-c", str(src), "-o",
                    str(tmp_path / "step.o")], check=True)


# Addresses that only the argument checks see: a call that they refuse reads nothing behind them.
CTX, X, OUT, OTHER = 1 << 20, 1 << 32, 1 << 36, 1 << 40
INF = float("inf")

ADJUST = dict(ctx=CTX, x=X, dtype=0, ldi=100, B=3, V=100, pen=None, per_row=0, hist=None, hist_off=None, prompt_len=None,
              bias_ids=None, bias=None, bias_off=None, mask=None, ldm=0, n_masks=0, mask_row=None, out=OUT, ldo=100, left=None,
              stream=None)
LOGPROBS = dict(ctx=CTX, x=X, dtype=0, ld=100, B=3, V=100, ids=OTHER, ldj=2, n=2, logprob=OUT, rank=None, lse=None, stream=None)
HEAD = dict(ctx=CTX, x=X, dtype=1, ldh=128, q=OTHER, ldq=64, scales=OTHER, scale_dtype=1, lds=4, zeros=None, ldz=0, group=32, B=3,
            V=100, D=128, out=OUT, ldl=100, stream=None)


def refused(fn, base, **change):
    lib = V.load_library()
    args = dict(base, **change)
    keep = args.get("pen")
    if isinstance(keep, V.Penalty):
        args["pen"] = ctypes.addressof(keep)
    assert getattr(lib, fn)(*args.values()) == -1, change
    return lib.vsmp_last_error().decode()


@pytest.mark.parametrize("change,words", [
    (dict(ctx=None), "null context"),
    (dict(x=None), "logits are required"),
    (dict(dtype=3), "dtype"),
    (dict(dtype=-1), "dtype"),
    (dict(B=0), "B >= 1"),
    (dict(V=0), "V >= 1"),
    (dict(V=(1 << 20) + 1, ldi=1 << 21, ldo=1 << 21), "vocabulary larger"),
    (dict(ldi=99), "stride"),
    (dict(ldi=1 << 62), "addressable"),
    (dict(x=X + 2), "aligned"),
    (dict(dtype=1, x=X + 1), "aligned"),
    (dict(out=None), "out is required"),
    (dict(out=OUT + 2), "out is required"),
    (dict(ldo=99), "ldo"),
    (dict(hist=OTHER), "hist and hist_off"),
    (dict(hist_off=OTHER), "hist and hist_off"),
    (dict(prompt_len=OTHER), "prompt_len"),
    (dict(bias_ids=OTHER), "bias"),
    (dict(bias=OTHER), "bias"),
    (dict(bias_ids=OTHER, bias_off=OTHER), "bias"),
    (dict(mask_row=OTHER), "need masks"),
    (dict(n_masks=2), "need masks"),
    (dict(mask=OTHER, n_masks=0, ldm=4), "n_masks >= 1"),
    (dict(mask=OTHER, n_masks=3, ldm=3), "ceil"),
    (dict(mask=OTHER, n_masks=2, ldm=4), "mask of its own"),
    (dict(pen=V.Penalty(repeat=0.0)), "repeat above 0"),
    (dict(pen=V.Penalty(repeat=-1.0)), "repeat above 0"),
    (dict(pen=V.Penalty(repeat=INF)), "finite"),
    (dict(pen=V.Penalty(presence=float("nan"))), "finite"),
    (dict(pen=V.Penalty(frequency=INF)), "finite"),
    (dict(out=X, ldo=104), "overlap"),
    (dict(out=X + 4), "overlap"),
    (dict(out=X, dtype=1), "overlap"),
    (dict(out=X + 4 * 299), "overlap"),
])
def test_adjust_refuses(change, words):
    assert words in refused("vsmp_adjust_logits", ADJUST, **change)


@pytest.mark.parametrize("change,words", [
    (dict(ctx=None), "null context"),
    (dict(x=None), "logits are required"),
    (dict(dtype=7), "dtype"),
    (dict(B=-1), "B >= 1"),
    (dict(V=(1 << 20) + 1, ld=1 << 21), "vocabulary larger"),
    (dict(ld=99), "stride"),
    (dict(n=-1), "0 <= n"),
    (dict(n=65, ldj=65), "0 <= n"),
    (dict(ids=None), "ids"),
    (dict(logprob=None), "logprob"),
    (dict(ldj=1), "ldj"),
    (dict(n=0), "lse is required"),
])
def test_logprobs_refuses(change, words):
    assert words in refused("vsmp_logprobs", LOGPROBS, **change)


@pytest.mark.parametrize("change,words", [
    (dict(ctx=None), "null context"),
    (dict(x=None), "required"),
    (dict(q=None), "required"),
    (dict(scales=None), "required"),
    (dict(out=None), "required"),
    (dict(dtype=0), "bf16 or f16"),
    (dict(scale_dtype=3), "scale dtype"),
    (dict(group=16), "group"),
    (dict(group=48), "group"),
    (dict(B=0), "B >= 1"),
    (dict(V=0), "V >= 1"),
    (dict(V=(1 << 20) + 1, ldl=1 << 21), "vocabulary larger"),
    (dict(D=0), "multiple of group"),
    (dict(D=48), "multiple of group"),
    (dict(D=16416, ldh=16416, ldq=8208, lds=513), "multiple of group"),
    (dict(D=96, group=64), "multiple of group"),
    (dict(ldh=120), "ldh"),
    (dict(ldh=129), "ldh"),
    (dict(x=X + 8), "16-byte"),
    (dict(ldq=48), "ldq"),
    (dict(ldq=72), "ldq"),
    (dict(q=OTHER + 8), "16-byte"),
    (dict(lds=3), "lds"),
    (dict(scales=OTHER + 1), "scales must be aligned"),
    (dict(zeros=OTHER, ldz=3), "ldz"),
    (dict(ldq=1 << 26), "2^26"),
    (dict(lds=1 << 24), "2^24"),
    (dict(zeros=OTHER, ldz=1 << 26), "2^26"),
    (dict(ldl=99), "ldl"),
    (dict(out=OUT + 2), "ldl"),
])
def test_head_refuses(change, words):
    assert words in refused("vsmp_head_logits_q4", HEAD, **change)


def test_bsampler_adjust_refuses_a_null_sampler():
    decode._lib()
    lib = V.load_library()
    assert lib.vsmp_bsampler_adjust_rows(None, X, 0, 100, 100, OTHER, 3, None, 0, None, None, None, None, None, 0, 0, None, OUT, 100,
                                         None, None) == -1
    assert "null sampler" in lib.vsmp_last_error().decode()


def test_python_refuses_host_tensors():
    import torch

    ctx = object.__new__(V.Context)  # no device here: the checks come before any call
    ctx._h, ctx.device = None, 0
    V.load_library()
    with pytest.raises(V.VsmpError, match="context's device"):
        ctx.adjust_logits(torch.zeros(2, 8))
    with pytest.raises(V.VsmpError, match="context's device"):
        ctx.logprobs(torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(V.VsmpError, match="context's device"):
        ctx.head_logits_q4(torch.zeros(2, 32).bfloat16(), torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1), 32)


def test_device_penalties_from_structs_and_arrays():
    rows = [V.Penalty(1.5, 0.25, -0.5, 7), V.Penalty()]
    a = V.to_device_penalties(rows, "cpu").numpy().view(V.PENALTY_DTYPE)
    assert a.tolist() == [(1.5, 0.25, -0.5, 7), (1.0, 0.0, 0.0, 0)]
    assert np.array_equal(V.to_device_penalties(a, "cpu").numpy().view(V.PENALTY_DTYPE), a)
