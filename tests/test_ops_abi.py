"""The operators' C ABI without a GPU: the argument structs the Python binding
packs have the C structs' layout, and arguments are refused before any device
is touched."""
import ctypes
import importlib
import os
import re
import struct
import subprocess

import pytest

from conftest import ROOT

STRUCTS = {"mx_layer_norm_args": "_NORM", "mx_layer_norm_backward_args": "_NORM_BACKWARD", "mx_dense_args": "_DENSE",
           "mx_dense_backward_args": "_DENSE_BACKWARD"}


@pytest.fixture(scope="module")
def ops():
    return importlib.import_module("maxim-rs_b200.ops")


def c_fields(name):
    text = open(os.path.join(ROOT, "include", "maxim_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
    fields = []
    for line in body.split(";"):
        if not line.strip():
            continue
        kind, names = re.match(r"\s*(?:const\s+)?(\w+\s*\**)\s*(.*)$", line, flags=re.S).groups()
        for n in names.split(","):
            fields.append(n.strip(" *\n"))
    return fields


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_packed_arguments_match_the_c_struct(ops, tmp_path, name):
    fields = c_fields(name)
    src = tmp_path / "layout.c"
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "maxim_b200.h"', "int main(void) {",
             '  printf("%%zu\\n", sizeof(%s));' % name]
    lines += ['  printf("%%zu %%zu\\n", offsetof(%s, %s), sizeof(((%s*)0)->%s));' % (name, f, name, f) for f in fields]
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    fmt = getattr(ops, STRUCTS[name])
    assert int(out[0]) == fmt.size
    codes = re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), fmt.format.lstrip("<"))
    assert len(codes) == len(fields)
    offset = 0
    for code, line in zip(codes, out[1:]):
        assert [offset, struct.calcsize("<" + code)] == [int(v) for v in line.split()]
        offset += struct.calcsize("<" + code)


def call(mx, entry, fmt, values):
    rc = getattr(mx.lib(), entry)(fmt.pack(*values), None)
    return rc, mx._native.last_error()


P = 1 << 20  # an address that is aligned to everything; never read


def norm(**kw):
    a = dict(x=P, scale=P, bias=P, y=P, mean=0, rstd=0, rows=4, c=8, xs=8, ys=8, dtype=0, pdtype=0, eps=1e-6, reserved=0)
    return list({**a, **kw}.values())


def norm_backward(**kw):
    a = dict(dy=P, x=P, scale=P, mean=P, rstd=P, dx=P, dscale=P, dbias=P, ws=0, ws_bytes=0, rows=4, c=8, dys=8, xs=8,
             dxs=8, dtype=0, pdtype=0)
    return list({**a, **kw}.values())


def dense(**kw):
    a = dict(x=P, w=P, bias=P, residual=0, y=P, pre=0, ws=0, ws_bytes=0, m=16, k=8, n=8, xs=8, ws_=8, rs=8, ys=8, ps=8,
             dtype=0, act=0, slope=0.2, reserved=0)
    return list({**a, **kw}.values())


def dense_backward(**kw):
    a = dict(dy=P, x=P, w=P, pre=0, dx=P, dw=P, db=P, ws=0, ws_bytes=0, m=16, k=8, n=8, dys=8, xs=8, ws_=8, ps=8, dxs=8,
             dws=8, dtype=0, act=0, slope=0.2, reserved=0)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("entry,layout,make,bad,message", [
    ("mx_layer_norm", "_NORM", norm, dict(dtype=3), "dtype 3"),
    ("mx_layer_norm", "_NORM", norm, dict(dtype=1, pdtype=2), "param_dtype"),
    ("mx_layer_norm", "_NORM", norm, dict(c=0), "c = 0"),
    ("mx_layer_norm", "_NORM", norm, dict(rows=-1), "rows = -1"),
    ("mx_layer_norm", "_NORM", norm, dict(x=0), "x is null"),
    ("mx_layer_norm", "_NORM", norm, dict(x=P + 2), "x is not aligned"),
    ("mx_layer_norm", "_NORM", norm, dict(scale=0), "scale is null"),
    ("mx_layer_norm", "_NORM", norm, dict(ys=7), "row stride of 7"),
    ("mx_layer_norm", "_NORM", norm, dict(eps=float("nan")), "eps"),
    ("mx_layer_norm_backward", "_NORM_BACKWARD", norm_backward, dict(mean=0), "mean is null"),
    ("mx_layer_norm_backward", "_NORM_BACKWARD", norm_backward, dict(dxs=3), "dx has a row stride"),
    ("mx_layer_norm_backward", "_NORM_BACKWARD", norm_backward, dict(dy=P + 1), "dy is not aligned"),
    ("mx_dense", "_DENSE", dense, dict(act=4), "act 4"),
    ("mx_dense", "_DENSE", dense, dict(k=0), "k = 0"),
    ("mx_dense", "_DENSE", dense, dict(n=1 << 31), "n = 2147483648"),
    ("mx_dense", "_DENSE", dense, dict(w=0), "w is null"),
    ("mx_dense", "_DENSE", dense, dict(residual=P, rs=1), "residual has a row stride"),
    ("mx_dense", "_DENSE", dense, dict(dtype=1, bias=P + 1), "bias is not aligned"),
    ("mx_dense_backward", "_DENSE_BACKWARD", dense_backward, dict(act=1), "pre is null"),
    ("mx_dense_backward", "_DENSE_BACKWARD", dense_backward, dict(x=0), "x is null"),
    ("mx_dense_backward", "_DENSE_BACKWARD", dense_backward, dict(w=0), "w is null"),
    ("mx_dense_backward", "_DENSE_BACKWARD", dense_backward, dict(dws=2), "dw has a row stride"),
])
def test_bad_arguments_are_refused(mx, ops, entry, layout, make, bad, message):
    rc, error = call(mx, entry, getattr(ops, layout), make(**bad))
    assert rc == mx._native.MX_E_INVALID
    assert entry in error and message in error, error


@pytest.mark.parametrize("entry", ["mx_layer_norm", "mx_layer_norm_backward", "mx_dense", "mx_dense_backward"])
def test_null_arguments_are_refused(mx, entry):
    assert getattr(mx.lib(), entry)(None, None) == mx._native.MX_E_INVALID
    if entry != "mx_layer_norm":
        assert getattr(mx.lib(), entry + "_workspace")(None, ctypes.byref(ctypes.c_int64())) == mx._native.MX_E_INVALID


def test_no_device_is_an_error(mx, ops):
    if mx.device_count() > 0:
        pytest.skip("a CUDA device is visible")
    for entry, layout, make in (("mx_layer_norm", ops._NORM, norm), ("mx_dense", ops._DENSE, dense)):
        rc, error = call(mx, entry, layout, make())
        assert rc not in (mx._native.MX_OK, mx._native.MX_E_INVALID) and error
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm(torch.zeros(2, 4), torch.ones(4), torch.ones(4))
