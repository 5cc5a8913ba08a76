"""The C interface of the gated block's operators on a host without a GPU: packed argument
structs, sizes and refusals.  No kernel runs: every call is host-only or fails validation."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from neurosim_gpu import block_ops, group_scaled, native, signal_ops

ROOT = Path(__file__).resolve().parents[1]
INCLUDE = ROOT / "include"


@pytest.fixture(scope="module")
def lib():
    return native.load_library()


def test_declared_symbols_are_exported(lib):
    names = re.findall(r"^\s*\w+\s+(ns_\w+)\s*\(", (INCLUDE / "neurosim_hip_block.h").read_text(),
                       flags=re.M)
    assert set(names) == {"ns_dropout", "ns_gated_forward", "ns_gated_backward",
                          "ns_gated_forward_bytes", "ns_gated_backward_bytes"}
    for name in (*names, "ns_recurrence_plan", "ns_recurrence_forward", "ns_recurrence_step",
                 "ns_recurrence_backward"):
        assert hasattr(lib, name), name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc is not installed")
def test_packed_structs_have_the_header_s_layout(tmp_path):
    """Sizes, and the place of each struct's last field, as a C compiler sees the headers."""
    source = tmp_path / "layout.c"
    source.write_text("""
#include <stddef.h>
#include <stdio.h>
#include "neurosim_hip_block.h"
int main(void) {
  printf("%zu %zu %zu\\n", sizeof(ns_gated_args), offsetof(ns_gated_args, workspace), offsetof(ns_gated_args, pre));
  printf("%zu %zu %zu\\n", sizeof(ns_dropout_args), offsetof(ns_dropout_args, offset), offsetof(ns_dropout_args, x));
  printf("%zu %zu %zu\\n", sizeof(ns_recurrence_args), offsetof(ns_recurrence_args, partials),
         offsetof(ns_recurrence_args, dy));
  return 0;
}
""")
    subprocess.run(["gcc", f"-I{INCLUDE}", str(source), "-o", str(tmp_path / "layout")], check=True)
    lines = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                           check=True).stdout.split("\n")
    gated, drop, recur = ([int(v) for v in line.split()] for line in lines[:3])
    assert gated == [block_ops._GATED.size, block_ops._GATED.size - 8, 32 + 4 * 16]
    assert drop == [block_ops._DROPOUT.size, block_ops._DROPOUT.size - 8, 16]
    assert recur[:2] == [signal_ops._RECUR.size, signal_ops._RECUR.size - 8]
    assert signal_ops._RECUR_FORWARD.size == recur[0] and recur[2] == recur[0] - 152


def plan(lib, *shape):
    sizes = (ctypes.c_int64 * 4)()
    fn = lib.ns_recurrence_plan
    fn.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int32, ctypes.c_void_p]
    code = fn(*shape, ctypes.addressof(sizes))
    return code, list(sizes)


def test_recurrence_plans(lib):
    """Tiles have 32 ticks.  Time is cut into chunks, of four whole tiles at least and none empty,
    only where workgroups are few and tiles many."""
    assert plan(lib, 2048, 8, 4096, 1) == (0, [1, 0, 64 * 8 * 4096, 8 * 4096])
    for ticks, batch, n, type in ((16384, 1, 2048, 1), (200, 1, 5, 0), (64, 1, 5, 0), (9000, 3, 64, 0),
                                  (0, 2, 4, 0), (700, 0, 4, 0), (40000, 1, 3, 2), (1000, 192, 3, 0),
                                  (1000, 191, 3, 0), (1000, 128, 129, 1), (767, 1, 4, 0), (704, 1, 4, 0)):
        code, (chunks, ends, kept, parts) = plan(lib, ticks, batch, n, type)
        tiles, lines = (ticks + 31) // 32, batch * n
        assert code == 0 and 1 <= chunks <= max(1, tiles // 4)
        if tiles < 24 or -(-n // 128) * batch >= 192:
            assert chunks == 1
        if chunks > 1:
            per = -(-tiles // chunks)
            assert (chunks - 1) * per < tiles
        assert ends == (2 * chunks * lines if chunks > 1 else 0)
        assert kept == tiles * lines and parts == chunks * lines
    assert plan(lib, 16384, 1, 2048, 1)[1][0] > 16 and plan(lib, 737, 1, 4, 0)[1][0] == 6
    for bad in ((-1, 1, 1, 0), (1, -1, 1, 0), (1, 1, 0, 0), (1, 1, 1, 9), (1 << 31, 1, 1, 0)):
        assert plan(lib, *bad)[0] != 0, bad


def message(lib, fn, args: bytes) -> str:
    fn = getattr(lib, fn)
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
    code = fn(args, None)
    lib.ns_last_error.restype = ctypes.c_char_p
    assert code != 0
    return lib.ns_last_error().decode()


def test_gated_refusals(lib):
    def args(rows=4, columns=8, width=16, type=0, activation=0, x=16, y=16, workspace=16, pre=0, dx=0):
        return block_ops._GATED.pack(rows, columns, width, type, activation, x, columns, 16, columns,
                                     16, columns, y, width, pre, 16, width, dx, 0, workspace)

    for change, text in ((dict(rows=-1), "negative"), (dict(type=7), "element type"),
                         (dict(activation=5), "activation"), (dict(columns=1 << 21), "at most"),
                         (dict(width=1 << 21), "at most"), (dict(x=0), "are required"),
                         (dict(y=0), "are required"),
                         (dict(rows=40, columns=7, workspace=0), "workspace"),
                         (dict(rows=40, columns=7, workspace=8), "workspace")):
        assert text in message(lib, "ns_gated_forward", args(**change)), change
    for change, text in ((dict(rows=0, dx=16), "at least one row"), (dict(dx=16), "forward's sums"),
                         (dict(rows=(1 << 21) + 1, dx=16), "at most 2097152 rows"),
                         (dict(dx=16, pre=16, workspace=0), "workspace")):
        assert text in message(lib, "ns_gated_backward", args(**change)), change


def test_gated_workspaces(lib):
    """Whole 16-byte rows at 16-byte addresses are read in place; others are laid out anew."""
    fn = lib.ns_gated_forward_bytes
    fn.restype, fn.argtypes = ctypes.c_int64, [ctypes.c_void_p]

    def bytes_(rows, columns, width, type, x=16, x_stride=None, gate_stride=None, up_stride=None):
        return fn(block_ops._GATED.pack(rows, columns, width, type, 0, x, x_stride or columns, 16,
                                        gate_stride or columns, 16, up_stride or columns, 16, width, 0,
                                        0, 0, 0, 0, 0))

    assert bytes_(40, 64, 30, 1) == 0
    assert bytes_(16, 63, 30, 1, x=18) == 0                        # few rows: read as they are
    assert bytes_(40, 64, 30, 1, x=24) == 40 * 128                 # 8 bytes off
    assert bytes_(40, 64, 30, 1, x_stride=68) == 40 * 128          # every other row off
    assert bytes_(40, 64, 30, 1, x_stride=72) == 0
    assert bytes_(40, 64, 30, 1, x_stride=8) == 40 * 128          # overlapping rows
    assert bytes_(40, 63, 30, 1) == (40 + 60) * 128
    assert bytes_(40, 64, 30, 1, gate_stride=72) == 60 * 128       # two strides
    assert bytes_(40, 64, 30, 1, x_stride=(1 << 22) + 8) == 40 * 128
    assert bytes_(40, 64, 30, 0) == 0 and bytes_(40, 65, 30, 0) == (40 + 60) * 272
    assert bytes_(5000, 1024, 320, 0) == (5000 + 640) * 32 * 192  # many in float32: in thirds
    assert bytes_(5000, 1025, 320, 0) == (5000 + 640) * 33 * 192
    assert bytes_(5000, 64, 320, 0) == 0 and bytes_(100, 8192, 3200, 0) == 0
    assert bytes_(0, 64, 30, 1) == 0


def test_dropout_refusals(lib):
    def args(count=4, type=0, threshold=10, x=16, out=16):
        return block_ops._DROPOUT.pack(count, type, threshold, x, 0, out, 0, 1, 2)

    for change, text in ((dict(count=-1), "negative"), (dict(type=3), "element type"),
                         (dict(threshold=-1), "threshold"), (dict(threshold=65537), "threshold"),
                         (dict(x=0), "required"), (dict(out=0), "required"),
                         (dict(count=1 << 62), "too large")):
        assert text in message(lib, "ns_dropout", args(**change)), change


def test_recurrence_refusals(lib):
    absent, present = (0, 0, 0), (16, 4, 4)

    def args(ticks=2, batch=1, channels=4, type=0, chunks=1, x=present, rates=16, y=present, z=absent,
             dz=absent, kept=0, dy=present, state=0, out_state=0, lengths=0, ends=0, work=16):
        return signal_ops._RECUR.pack(ticks, batch, channels, type, chunks, *x, *present, *present, *z,
                                      *y, rates, state, out_state, lengths, kept, ends, *dy, 0, *present,
                                      *present, *present, *dz, 0, work, work)

    for change, text in ((dict(ticks=-1), "N > 0"), (dict(channels=0), "N > 0"),
                         (dict(type=4), "element type"), (dict(chunks=0), "one chunk"),
                         (dict(rates=0), "rates"), (dict(x=absent), "required"),
                         (dict(y=absent), "output"), (dict(ticks=200, chunks=2), "workspace"),
                         (dict(batch=1 << 30, channels=1 << 30), "too large")):
        assert text in message(lib, "ns_recurrence_forward", args(**change)), change
    for change, text in ((dict(), "one tick"), (dict(ticks=1, lengths=16), "one tick"),
                         (dict(ticks=1), "in place"), (dict(ticks=1, state=16, out_state=32), "in place")):
        assert text in message(lib, "ns_recurrence_step", args(**change)), change
    for change, text in ((dict(ticks=0), "at least one tick"), (dict(), "forward's states"),
                         (dict(kept=16, dy=absent), "required"), (dict(kept=16, work=0), "required"),
                         (dict(kept=16, z=present), "dz is given"),
                         (dict(kept=16, ticks=200, chunks=2), "workspace")):
        assert text in message(lib, "ns_recurrence_backward", args(**change)), change


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc is not installed")
def test_packed_4_bit_structs_have_the_header_s_layout(tmp_path):
    source = tmp_path / "layout.c"
    source.write_text("""
#include <stddef.h>
#include <stdio.h>
#include "neurosim_hip_q4.h"
int main(void) {
  printf("%zu %zu\\n", sizeof(ns_q4_matrix), offsetof(ns_q4_matrix, scale_type));
  printf("%zu %zu %zu\\n", sizeof(ns_q4_product_args), offsetof(ns_q4_product_args, workspace),
         offsetof(ns_q4_product_args, type));
  return 0;
}
""")
    subprocess.run(["gcc", f"-I{INCLUDE}", str(source), "-o", str(tmp_path / "layout")], check=True)
    lines = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                           check=True).stdout.split("\n")
    matrix, product = ([int(v) for v in line.split()] for line in lines[:2])
    assert matrix == [group_scaled._MATRIX.size, 48]
    assert product == [group_scaled._PRODUCT.size, group_scaled._PRODUCT.size - 8,
                       group_scaled._PRODUCT.size - 16]


def test_4_bit_refusals(lib):
    def matrix(rows=4, columns=64, group=32, codes=16, scales=16, scale_type=1):
        return rows, columns, group, codes, scales, 0, scale_type

    def product(m=2, x=16, out=16, type=0, **more):
        return group_scaled._PRODUCT.pack(*matrix(**more), m, x, 64, 0, out, 4, type, 0)

    changes = ((dict(rows=-1), "negative"), (dict(columns=(1 << 23) + 1), "at most"),
               (dict(group=16), "32, 64"), (dict(group=192), "32, 64"), (dict(group=1 << 39), "up to"),
               (dict(group=(1 << 23) + 128), "up to"), (dict(codes=0), "required"),
               (dict(scales=0), "required"), (dict(codes=8), "aligned"), (dict(scale_type=9), "scales"))
    for change, text in changes:
        assert text in message(lib, "ns_q4_product", product(**change)), change
        for fn in (lib.ns_q4_quantize, lib.ns_q4_dequantize):
            fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64,
                                                     ctypes.c_int32, ctypes.c_void_p]
            assert fn(group_scaled._MATRIX.pack(*matrix(**change)), 16, 64, 0, None) != 0
            assert text in lib.ns_last_error().decode(), change
    for change, text in ((dict(m=-1), "negative"), (dict(x=0), "required"), (dict(out=0), "required"),
                         (dict(type=5), "element type"), (dict(columns=50_000, rows=100), "workspace")):
        assert text in message(lib, "ns_q4_product", product(**change)), change


def test_4_bit_workspaces(lib):
    """Workgroups share K, and need a workspace, only where the weight's rows are few."""
    fn = lib.ns_q4_product_floats
    fn.restype, fn.argtypes = ctypes.c_int64, [ctypes.c_int64] * 3 + [ctypes.c_int32]
    assert fn(1, 50_000, 1024, 0) == 0 and fn(0, 5, 5, 0) == 0 and fn(5, 0, 5, 0) == 0
    assert fn(33, 1000, 50_000, 1) % (33 * 1000) == 0 and fn(33, 1000, 50_000, 1) > 33 * 1000
