"""What the launchers in paged.c ask of the device, with the launch replaced by one that writes it down: no device, no
kernel.  Each check runs in a process of its own, under a time limit (a launcher that never returns fails its test)."""
import ctypes as ct
import json
import os
import shutil
import subprocess
import sys

import pytest

import test_paged_args as args

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "switch-l4t-gpu_amd", "csrc")
MOST = 2**32 - 1                                        # work items of a launch's grid
TREE, JOIN, LOGITS = 12, 36, 39                         # first kernels of each kind in paged.c's table

STUB = """
#include <string.h>
#include "sgpu_internal.h"
int launches, kernels[1024];
unsigned blocks_of[1024], threads_of[1024];
unsigned char args_of[1024][160];
int sgpu_internal_paged_launch(int kernel, unsigned blocks, unsigned threads, void **args, void *stream) {
    (void)stream;
    if (launches == 1024) return -99;
    kernels[launches] = kernel;
    blocks_of[launches] = blocks;
    threads_of[launches] = threads;
    if (kernel >= SGPU_PG_LOGITS) memcpy(args_of[launches], args[0], 160);
    launches++;
    return 0;
}
"""


@pytest.fixture(scope="module")
def stubbed(tmp_path_factory):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("no C compiler")
    d = tmp_path_factory.mktemp("paged")
    (d / "stub.c").write_text(STUB)
    lib = str(d / "libpaged.so")
    subprocess.run([gcc, "-O1", "-fPIC", "-shared", "-std=gnu11", "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-I", "/opt/rocm/include",
                    os.path.join(CSRC, "paged.c"), str(d / "stub.c"), "-o", lib, "-lm"], check=True)
    return lib


def child(lib, kind, kw, half):
    """One call; its status, the workspace it asks for, and its launches."""
    import sgpu

    L = ct.CDLL(lib)
    a = {"tree": args.tree, "append": args.append, "logits": args.logits}[kind](sgpu, **kw)
    need = 0
    if kind == "tree":
        L.sgpu_attn_tree_workspace.restype = ct.c_size_t
        need = L.sgpu_attn_tree_workspace(ct.byref(a))
        rc = getattr(L, "sgpu_attn_tree" + half)(ct.byref(a), ct.c_void_p(args.P), ct.c_size_t(need), None)
    else:
        rc = getattr(L, {"append": "sgpu_kv_append", "logits": "sgpu_logits_adjust"}[kind] + half)(ct.byref(a), None)
    n = ct.c_int.in_dll(L, "launches").value
    of = {k: list((t * 1024).in_dll(L, k))[:n] for k, t in (("kernels", ct.c_int), ("blocks_of", ct.c_uint), ("threads_of", ct.c_uint))}
    raw = ((ct.c_ubyte * 160) * 1024).in_dll(L, "args_of")
    print(json.dumps({"rc": rc, "need": need, "launches": list(zip(of["kernels"], of["blocks_of"], of["threads_of"])),
                      "args": [bytes(raw[i]).hex() for i in range(n)]}))


def call(lib, kind, half="", **kw):
    p = subprocess.run([sys.executable, os.path.abspath(__file__), lib, kind, half, json.dumps(kw)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stderr
    got = json.loads(p.stdout)
    assert got["rc"] == 0
    for kernel, blocks, threads in got["launches"]:
        assert 0 < blocks and blocks * threads <= MOST, (kernel, blocks, threads)
    return got


class LogitsPart(ct.Structure):
    """paged_logits, as the kernel takes it."""

    _fields_ = ([(n, ct.c_void_p) for n in ("x", "y", "tok", "span", "bias_id", "bias_span", "rep", "freq", "pres", "bias", "allow")] +
                [(n, ct.c_longlong) for n in ("x_row", "y_row", "allow_row")] +
                [(n, ct.c_int) for n in ("rows", "V", "n_tok", "n_bias", "C", "groups")])


@pytest.mark.parametrize("half", ["", "_h"])
@pytest.mark.parametrize("rows,V,allow_row,bias", [(1, 1000, 32, True), (512, 151936, 4748, True), (513, 8193, 257, False), ((1 << 22) - 1, 8, 1, True),
                                                   (1 << 22, 8, 1, True), (5_000_011, 6, 0, True), ((1 << 24) - 1, 100, 4, True),
                                                   ((1 << 24) - 1, 1 << 20, 1 << 15, False)])
def test_logits_of_any_number_of_rows(stubbed, rows, V, allow_row, bias, half):
    """Every row once, each launch with its rows' parts of the tables, whatever the rows' number."""
    P, optional = args.P, {} if bias else dict(bias_span=None, rep=None, pres=None)
    got = call(stubbed, "logits", half, rows=rows, V=V, x_row=V + 8, y_row=V, allow_row=allow_row, **optional)
    first, size = 0, 2 if half else 4
    for (kernel, blocks, _), raw in zip(got["launches"], got["args"]):
        a = LogitsPart.from_buffer_copy(bytes.fromhex(raw)[:ct.sizeof(LogitsPart)])
        assert kernel == LOGITS + 2 * bias + bool(half) and blocks == a.rows * a.groups and (a.V, a.x_row, a.y_row) == (V, V + 8, V)
        assert (a.x, a.y, a.allow) == (P + size * first * (V + 8), 2 * P + size * first * V, 11 * P + 4 * first * allow_row)
        assert (a.tok, a.span, a.freq) == (3 * P, 4 * P + 16 * first, 6 * P + 4 * first)
        assert (a.rep, a.pres, a.bias_span) == ((5 * P + 4 * first, 7 * P + 4 * first, 10 * P + 8 * first) if bias else (None,) * 3)
        assert (a.n_tok, a.n_bias, a.allow_row) == (10, 4, allow_row) and (a.bias_id, a.bias) == (8 * P, 9 * P)
        first += a.rows
    assert first == rows


@pytest.mark.parametrize("half", ["", "_h"])
@pytest.mark.parametrize("kw", [
    dict(B=4096, NKV=8, NH=8, R=(1 << 23) - 1, max_q=1 << 20, max_kv=640, table_pages=40, table_row=40),     # more row tiles than a grid
    dict(B=1 << 19, NKV=8, NH=8, R=1 << 22, max_q=1024, max_kv=128, table_pages=8, table_row=8),
    dict(B=(1 << 23) - 1, NKV=1, NH=1, R=1 << 23, max_q=1 << 20, max_kv=128, table_pages=8, table_row=8),
    dict(B=1, NKV=1, NH=1, R=(1 << 26) - 1, max_q=1 << 26, max_kv=128, table_pages=8, table_row=8),
    dict(B=2, NKV=1, NH=1, R=(1 << 26) - 1, max_q=1, max_kv=100000, table_pages=6250, table_row=6250),       # more rows to join
    dict(B=2, NKV=1, NH=3, R=((1 << 26) - 1) // 3, max_q=40, max_kv=100000, table_pages=6250, table_row=6250),
    dict(B=64, max_kv=4096, table_pages=256, table_row=256)], ids=lambda kw: ",".join(f"{k}={v}" for k, v in kw.items()))
def test_attention_fits_a_grid(stubbed, kw, half):
    """Hints and rows as many as the call allows: each launch fits a grid."""
    got = call(stubbed, "tree", half, pages=7000, mask=None, q_row=1 << 20, out_row=1 << 20, kv_row=1024, page_stride=1 << 14, **kw)
    assert TREE <= got["launches"][0][0] < JOIN and len(got["launches"]) in (1, 2)


@pytest.mark.parametrize("half", ["", "_h"])
@pytest.mark.parametrize("page", [1 << 30, (1 << 30) + 1, 2**31 - 1])
def test_pages_of_any_size_without_a_table(stubbed, page, half):
    """A table without entries allows any page size: the calls return."""
    for pages in (0, 3):
        for kind in ("tree", "append"):
            got = call(stubbed, kind, half, pages=pages, table_pages=0, table_row=0, page=page)
            assert len(got["launches"]) >= 1


if __name__ == "__main__":
    for p in (os.path.join(ROOT, "switch-l4t-gpu_amd"), os.path.dirname(os.path.abspath(__file__))):
        sys.path.insert(0, p)
    child(sys.argv[1], sys.argv[2], json.loads(sys.argv[4]), sys.argv[3])
