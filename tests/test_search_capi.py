"""Beams and the states behind them on the CPU: every declared entry point is exported, the header compiles as C, the
structs have their layout, and bad arguments are refused with a message before any GPU work. No GPU calls."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest

import verbo_amd as V

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "vsmp_beam.h"


def test_entry_points_are_declared_and_exported():
    names = re.findall(r"VSMP_API\s+[\w\s\*]+?\b(vsmp_\w+)\s*\(", HEADER.read_text())
    assert names == ["vsmp_beam_select", "vsmp_reorder_rows", "vsmp_pages_step", "vsmp_pages_compact"]
    lib = V.load_library()
    for n in names:
        assert hasattr(lib, n), n


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc absent")
def test_header_compiles_as_c_and_the_structs_have_their_layout(tmp_path):
    src = tmp_path / "h.c"
    lines = ["#include <stddef.h>", "#include \"vsmp_beam.h\""]
    for c, py in (("vsmp_planes", V._PlanesArg), ("vsmp_pages", V._PagesArg)):
        lines.append(f"_Static_assert(sizeof({c}) == {ctypes.sizeof(py)}, \"size\");")
        lines += [f"_Static_assert(offsetof({c}, {f[0]}) == {getattr(py, f[0]).offset}, \"{f[0]}\");" for f in py._fields_]
    src.write_text("\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"), "-c", str(src), "-o",
                    str(tmp_path / "h.o")], check=True)


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ absent")
def test_the_documented_step_compiles(tmp_path):
    """The C++ block that INTEGRATION.md shows for these calls, with the variables that it names."""
    block = [b for b in re.findall(r"```cpp\n(.*?)```", (ROOT / "INTEGRATION.md").read_text(), re.S) if "vsmp_beam.h" in b]
    assert len(block) == 1
    body = "\n".join(line for line in block[0].splitlines() if not line.startswith("#include"))
    src = tmp_path / "step.cpp"
    src.write_text("""#include "vsmp_beam.h"
void step(vsmp_ctx* ctx, const void* d_logits, long long ld, int G, int W, int V, const float* d_scores, const int* stops, int n_stop,
          int* d_token, int* d_parent, float* d_score, int* d_end_token, int* d_end_parent, float* d_end_score, int* d_n_end,
          void* const* d_planes, int n_planes, long long row_stride, int heads, long long piece_stride, int room, int token_bytes,
          int* d_lens, void* const* d_pools, int n_pages, int page_tokens, int row_pages, int* d_table, int* d_ref,
          int* d_next_table, int* d_next_lens, int* d_next_ref, int* d_ok, void* stream) {
""" + body + "\n}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"), "-c", str(src), "-o",
                    str(tmp_path / "step.o")], check=True)


# Addresses that only the argument checks see: a call that they refuse reads nothing behind them.
CTX, X, A, B, C, D, E, F = (1 << 20, *(k << 34 for k in range(1, 8)))


def refused(fn, *args):
    lib = V.load_library()
    assert getattr(lib, fn)(*args) == -1
    return lib.vsmp_last_error().decode()


SELECT = dict(ctx=CTX, x=X, dtype=0, ld=100, G=2, W=3, V=100, scores=A, N=3, stops=None, n_stop=0, token=B, parent=C, score=D,
              end_token=None, end_parent=None, end_score=None, n_end=None, stream=None)


@pytest.mark.parametrize("change,words", [
    (dict(ctx=None), "null context"),
    (dict(x=None), "logits and scores"),
    (dict(scores=None), "logits and scores"),
    (dict(dtype=3), "dtype"),
    (dict(dtype=-1), "dtype"),
    (dict(G=0), ">= 1"),
    (dict(W=0), ">= 1"),
    (dict(V=0), ">= 1"),
    (dict(N=0), ">= 1"),
    (dict(W=65), "at most 64"),
    (dict(N=65), "at most 64"),
    (dict(V=(1 << 20) + 1, ld=1 << 21), "vocabulary larger"),
    (dict(G=1 << 30, W=64), "beams"),
    (dict(ld=99), "stride"),
    (dict(ld=1 << 60), "addressable"),
    (dict(x=X + 2), "aligned"),
    (dict(dtype=2, x=X + 1), "aligned"),
    (dict(scores=A + 2), "aligned"),
    (dict(n_stop=-1), "n_stop"),
    (dict(n_stop=17), "n_stop"),
    (dict(n_stop=2), "n_stop"),
    (dict(token=None), "token, parent and score"),
    (dict(score=None), "token, parent and score"),
    (dict(end_token=E), "go together"),
    (dict(end_token=E, end_parent=E, end_score=E), "go together"),
    (dict(n_end=E), "go together"),
    (dict(token=B + 2), "outputs must be aligned"),
    (dict(score=D + 1), "outputs must be aligned"),
    (dict(end_token=E, end_parent=E, end_score=E, n_end=E + 2), "outputs must be aligned"),
])
def test_select_refuses(change, words):
    assert words in refused("vsmp_beam_select", *dict(SELECT, **change).values())


def planes(**change):
    return V._PlanesArg(**dict(dict(planes=A, n_planes=2, rows=12, row_stride=4096, pieces=2, piece_stride=2048, tokens=16, token_bytes=128), **change))


def pages(at, **change):
    return V._PagesArg(**dict(dict(rows=4, row_pages=8, n_pages=12, page_tokens=16, table=at, ldt=8, lens=at + 4096, ref=at + 8192), **change))


PLANES_REFUSED = [
    (dict(planes=None), "array of addresses"),
    (dict(planes=A + 4), "array of addresses"),
    (dict(n_planes=0), "at least one"),
    (dict(rows=0), "at least one"),
    (dict(pieces=0), "at least one"),
    (dict(tokens=0), "at least one"),
    (dict(token_bytes=0), "at least one"),
    (dict(token_bytes=1 << 28, piece_stride=1 << 33, row_stride=1 << 34), "2^31"),
    (dict(pieces=1 << 28), "2^34"),
    (dict(row_stride=-4096), "strides"),
    (dict(piece_stride=-2048), "strides"),
    (dict(row_stride=1 << 62), "strides"),
    (dict(row_stride=4095), "overlap"),
    (dict(piece_stride=2047), "overlap"),
    (dict(row_stride=2048, piece_stride=12 * 2048 - 1), "overlap"),
]


@pytest.mark.parametrize("change,words", PLANES_REFUSED)
def test_planes_are_checked(change, words):
    p = planes(**change)
    assert words in refused("vsmp_reorder_rows", CTX, ctypes.addressof(p), B, 4, None, None)


def test_reorder_refuses():
    p = planes()
    at = ctypes.addressof(p)
    assert "null context" in refused("vsmp_reorder_rows", None, at, B, 4, None, None)
    assert "planes and parent" in refused("vsmp_reorder_rows", CTX, None, B, 4, None, None)
    assert "planes and parent" in refused("vsmp_reorder_rows", CTX, at, None, 4, None, None)
    for width in (0, 5, 65):
        assert "width" in refused("vsmp_reorder_rows", CTX, at, B, width, None, None)
    assert "aligned" in refused("vsmp_reorder_rows", CTX, at, B + 2, 4, None, None)
    assert "aligned" in refused("vsmp_reorder_rows", CTX, at, B, 4, C + 1, None)


PAGES_REFUSED = [
    (dict(rows=0), dict(), "rows"),
    (dict(), dict(rows=8193), "rows"),
    (dict(n_pages=0), dict(n_pages=0), "n_pages"),
    (dict(n_pages=(1 << 20) + 1), dict(), "n_pages"),
    (dict(row_pages=0), dict(), "row_pages"),
    (dict(page_tokens=0), dict(), "page_tokens"),
    (dict(), dict(row_pages=1 << 27, ldt=1 << 27), "2^30"),
    (dict(table=None), dict(), "required"),
    (dict(lens=None), dict(), "required"),
    (dict(), dict(ref=None), "required"),
    (dict(table=C + 2), dict(), "aligned"),
    (dict(), dict(lens=D + 4097), "aligned"),
    (dict(ldt=7), dict(), "ldt"),
    (dict(), dict(ldt=1 << 62), "ldt"),
    (dict(), dict(n_pages=13), "same pool"),
    (dict(), dict(page_tokens=8, row_pages=16, ldt=16), "same pool"),
    (dict(), dict(row_pages=7), "room"),
    (dict(), dict(table=C), "must not overlap"),
    (dict(), dict(ref=C + 8192 + 44), "must not overlap"),
    (dict(), dict(lens=C + 4 * 31), "must not overlap"),
    (dict(), dict(lens=D + 4 * 31), "to's arrays"),
]


@pytest.mark.parametrize("a,b,words", PAGES_REFUSED)
def test_pages_are_checked(a, b, words):
    x, y = pages(C, **a), pages(D, **b)
    assert words in refused("vsmp_pages_step", CTX, ctypes.addressof(x), ctypes.addressof(y), None, None, 1, None, None, None)
    assert words in refused("vsmp_pages_compact", CTX, ctypes.addressof(x), ctypes.addressof(y), None, None, None, None)


def test_steps_refuse():
    x, y, p = pages(C), pages(D), planes()
    ax, ay, ap = ctypes.addressof(x), ctypes.addressof(y), ctypes.addressof(p)
    assert "null context" in refused("vsmp_pages_step", None, ax, ay, None, None, 1, None, None, None)
    assert "null context" in refused("vsmp_pages_compact", None, ax, ay, None, None, None, None)
    assert "from and to" in refused("vsmp_pages_step", CTX, None, ay, None, None, 1, None, None, None)
    assert "from and to" in refused("vsmp_pages_compact", CTX, ax, None, None, None, None, None)
    for k in (3, 4, 7):
        args = [CTX, ax, ay, None, None, 1, None, None, None]
        args[k] = E + 2
        assert "aligned" in refused("vsmp_pages_step", *args)
    for k in (4, 5):
        args = [CTX, ax, ay, ap, None, None, None]
        args[k] = E + 2
        assert "aligned" in refused("vsmp_pages_compact", *args)
    q = planes(n_planes=1 << 16, rows=1 << 18, tokens=16)
    big = [pages(at << 4, n_pages=1 << 18, lens=(at << 4) + (1 << 24), ref=(at << 4) + (1 << 25)) for at in (C, D)]
    for fn, rest in (("vsmp_pages_step", (None, None, 1, ctypes.addressof(q), None, None)), ("vsmp_pages_compact", (ctypes.addressof(q), None, None, None))):
        assert "too many planes" in refused(fn, CTX, ctypes.addressof(big[0]), ctypes.addressof(big[1]), *rest)
    z = pages(D, rows=5)
    assert "same rows" in refused("vsmp_pages_compact", CTX, ax, ctypes.addressof(z), None, None, None, None)
    for change, words in PLANES_REFUSED + [(dict(rows=11), "n_pages rows"), (dict(tokens=15), "n_pages rows"), (dict(rows=13), "n_pages rows")]:
        q = planes(**change)
        if change.get("rows") == 0 or change.get("tokens") == 0:
            words = "at least one"
        assert words in refused("vsmp_pages_step", CTX, ax, ay, None, None, 1, ctypes.addressof(q), None, None), change
        assert words in refused("vsmp_pages_compact", CTX, ax, ay, ctypes.addressof(q), None, None, None), change


def test_python_refuses_before_the_call():
    """Tensors that are not the device's, of another type or too short, without a GPU: on the CPU they are all of that."""
    import torch

    x = torch.zeros(4, 10)
    for make in (lambda: V.Planes([x]), lambda: V.Planes([]), lambda: V.Pages(torch.zeros(2, 2, dtype=torch.int32), x, x, 4)):
        with pytest.raises(V.VsmpError):
            make()
