"""The block operators' C entries without a GPU: what they refuse before touching the device,
and the host's check for overlapping outputs."""
import ctypes
import shutil
import subprocess

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def lib(scb):
    return scb.load_library()


def refused(lib, rc, words):
    assert rc == -1
    msg = lib.scb_last_error(None).decode()
    assert words in msg, msg


def norm(lib, **kw):
    a = dict(x=16, sn=80, sl=8, dtype=0, n=2, l=10, c=8, groups=2, w=None, b=None, eps=1e-5, act=0, y=16, yn=80, yl=8)
    a.update(kw)
    return lib.scb_group_norm(a["x"], a["sn"], a["sl"], a["dtype"], a["n"], a["l"], a["c"], a["groups"], a["w"], a["b"],
                              a["eps"], a["act"], a["y"], a["yn"], a["yl"], None, None, None, 0, None)


@pytest.mark.parametrize("change,words", [
    (dict(dtype=1), "element type"), (dict(n=-1), "negative"), (dict(c=0), "positive"), (dict(groups=3), "3 groups"),
    (dict(groups=0), "0 groups"), (dict(act=4), "activation"), (dict(x=None), "NULL"), (dict(sl=-8), "negative"),
    (dict(yl=7), "overlapping"), (dict(yn=0), "overlapping"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
])
def test_group_norm_refuses(lib, change, words):
    refused(lib, norm(lib, **change), words)


def test_group_norm_nothing_to_do(lib):
    assert norm(lib, n=0) == 0


def rotate(lib, scb, **kw):
    a = dict(dtype=0, b=1, l=4, d=16, pos=16, pos_dtype=4, freq=16, sections=(4, 4), layout=0, x=16, y=16, heads=2,
             yh=16, sl=32)
    a.update(kw)
    q = scb.backend.ScbHeads(a["x"], a["y"], a["heads"], 0, 32, 16, 0, a["sl"], a["yh"])
    n = len(a["sections"])
    return lib.scb_rotate_axes(q, None, a["dtype"], a["b"], a["l"], a["d"], a["pos"], a["pos_dtype"], 0, n, 1, a["freq"],
                               (ctypes.c_int * n)(*a["sections"]), n, a["layout"], 0, None)


@pytest.mark.parametrize("change,words", [
    (dict(dtype=7), "element type"), (dict(d=1), "at least 2"), (dict(sections=(4, 5)), "pairs"),
    (dict(sections=(0,)), "pairs"), (dict(sections=(-1, 4)), "section"), (dict(sections=(1,) * 5), "axes"),
    (dict(layout=3), "layout"), (dict(pos_dtype=2), "positions"), (dict(pos=None), "NULL"), (dict(freq=None), "NULL"),
    (dict(x=None), "NULL"), (dict(pos=18), "misaligned"), (dict(x=18), "aligned"), (dict(yh=8), "overlapping"),
    (dict(sl=16), "overlapping"), (dict(heads=-1), "heads"),
])
def test_rotate_axes_refuses(lib, scb, change, words):
    refused(lib, rotate(lib, scb, **change), words)


def attend(lib, scb, **kw):
    a = dict(dtype=2, b=1, lq=3, lk=4, h=4, hk=2, d=16, scale=1.0, q=16, k=16, o=16, ol=64)
    a.update(kw)
    rows = [scb.backend.ScbRows(p, 0, s, 16) for p, s in ((a["q"], 64), (a["k"], 32), (16, 32), (a["o"], a["ol"]))]
    return lib.scb_attention(*rows, a["dtype"], a["b"], a["lq"], a["lk"], a["h"], a["hk"], a["d"], None, 0, a["scale"],
                             None, 0, None)


@pytest.mark.parametrize("change,words", [
    (dict(dtype=0), "element type"), (dict(lq=-1), "negative"), (dict(hk=3), "share"), (dict(h=0), "share"),
    (dict(d=257), "256"), (dict(d=0), "256"), (dict(scale=float("inf")), "finite"), (dict(q=None), "NULL"),
    (dict(k=None), "NULL"), (dict(q=17), "aligned"), (dict(ol=32), "overlapping"),
])
def test_attention_refuses(lib, scb, change, words):
    refused(lib, attend(lib, scb, **change), words)


def test_attention_nothing_to_do(lib, scb):
    assert attend(lib, scb, lq=0) == 0 and attend(lib, scb, b=0) == 0


def test_workspace_calls(lib):
    need = ctypes.c_size_t(7)
    refused(lib, lib.scb_group_norm_workspace(1, 1, 6, 4, ctypes.byref(need)), "4 groups")
    assert need.value == 0
    assert lib.scb_group_norm_workspace(0, 5, 8, 2, ctypes.byref(need)) == 0 and need.value == 0
    refused(lib, lib.scb_attention_workspace(1, 1, 1, 3, 2, 8, ctypes.byref(need)), "sizes")
    assert lib.scb_attention_workspace(1, 5, 0, 4, 2, 8, ctypes.byref(need)) == 0 and need.value == 0


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_distinct_elements(tmp_path):
    """Outputs whose elements coincide are found whatever the order of their dimensions."""
    src = tmp_path / "distinct.cpp"
    src.write_text("""
#include "host_logic.h"
#include <cstdio>
using namespace scb;
#define CHECK(c) do { if (!(c)) { printf("FAILED line %d\\n", __LINE__); return 1; } } while (0)
int main() {
  CHECK(distinct_elements(8, {{4, 8}, {3, 32}}));
  CHECK(distinct_elements(8, {{3, 32}, {4, 8}}));
  CHECK(distinct_elements(8, {{4, 100}, {3, 8}, {5, 500}}));
  CHECK(!distinct_elements(8, {{4, 7}, {3, 32}}));
  CHECK(!distinct_elements(8, {{4, 8}, {3, 31}}));
  CHECK(!distinct_elements(8, {{4, 0}, {3, 32}}));
  CHECK(distinct_elements(8, {{1, 0}, {3, 8}}));
  CHECK(distinct_elements(8, {{0, 0}, {3, 1}}));
  CHECK(!distinct_elements(16, {{2, 64}, {4, 16}, {2, 48}}));
  CHECK(distinct_elements(1, {{1 << 20, int64_t(1) << 31}, {2, int64_t(1) << 52}}));
  printf("ok\\n");
}
""")
    exe = tmp_path / "distinct"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{ROOT / 'scunet-rs_b200' / 'csrc'}", str(src),
                    "-o", str(exe)], check=True, capture_output=True, timeout=120)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "ok\n"
