"""Host side of a layer's norms and products: struct layouts and the refusals that need no device (CPU)."""
import ctypes
import os
import subprocess

import pytest

from mimir_framework_b200 import abi, runtime as rt

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header(tmp_path):
    lines, want = [], []
    for name in ("MimirNormRows", "MimirLinear"):
        cls = getattr(abi, name)
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu ", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
        lines.append(f'printf("%zu ", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mimir_b200.h"\nint main(void) {' + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


NORM = dict(x=16, y=32, rows=4, n=64, type=abi.T_BF16, y_type=abi.T_BF16, x_stride=64, y_stride=64)
LINEAR = dict(x=16, w=32, out=48, rows=4, n_in=64, n_out=40, type=abi.T_BF16, out_type=abi.T_F32, x_stride=64, w_stride=64, out_stride=40)
GATED = LINEAR | dict(up=64, up_stride=64)
CODED = LINEAR | dict(type=abi.T_E4M3, x_scale=4, w_scale=4)


def refused(call, args, change, status):
    make = rt.norm_rows if call is rt.dev_norm_rows else rt.linear
    with pytest.raises(rt.MimirB200Error) as e:
        call(make(**(args | change)))
    assert e.value.status == status, e.value


@pytest.mark.parametrize("change,status", [
    (dict(type=abi.T_E4M3), abi.E_INVALID), (dict(type=9), abi.E_INVALID), (dict(y_type=-1), abi.E_INVALID), (dict(y_type=abi.T_I8), abi.E_UNSUPPORTED),
    (dict(rows=-1), abi.E_INVALID), (dict(n=0), abi.E_INVALID), (dict(n=32769, x_stride=40000, y_stride=40000), abi.E_UNSUPPORTED), (dict(eps=-1.0), abi.E_INVALID),
    (dict(eps=float("nan")), abi.E_INVALID), (dict(eps=float("inf")), abi.E_INVALID), (dict(norm=False, gamma=4), abi.E_INVALID), (dict(y_type=abi.T_E4M3), abi.E_INVALID),
    (dict(y_scale=4), abi.E_INVALID), (dict(x_stride=63), abi.E_INVALID), (dict(y_stride=-64), abi.E_INVALID), (dict(residual=64, residual_stride=8), abi.E_INVALID),
    (dict(sum=64, sum_stride=0), abi.E_INVALID), (dict(sum=32, sum_stride=64), abi.E_INVALID), (dict(sum=16, sum_stride=72), abi.E_INVALID),
    (dict(y=16, y_stride=72), abi.E_INVALID), (dict(y=16, y_type=abi.T_F16), abi.E_INVALID), (dict(x_stride=1 << 36), abi.E_INVALID)])
def test_norm_rows_refuses(change, status):
    refused(rt.dev_norm_rows, NORM, change, status)


@pytest.mark.parametrize("change,status", [
    (dict(type=abi.T_F32), abi.E_UNSUPPORTED), (dict(type=abi.T_I8), abi.E_UNSUPPORTED), (dict(type=7), abi.E_INVALID), (dict(out_type=abi.T_E4M3), abi.E_INVALID),
    (dict(rows=-1), abi.E_INVALID), (dict(n_in=0), abi.E_INVALID), (dict(n_out=-3), abi.E_INVALID), (dict(activation=0), abi.E_UNSUPPORTED),
    (dict(activation=abi.ELT_MISH), abi.E_UNSUPPORTED), (dict(activation=-2), abi.E_UNSUPPORTED), (dict(x_scale=4), abi.E_INVALID), (dict(w_scale=4), abi.E_INVALID),
    (dict(up_scale=4), abi.E_INVALID), (dict(x_stride=60), abi.E_INVALID), (dict(x_stride=68), abi.E_UNSUPPORTED), (dict(w_stride=65), abi.E_UNSUPPORTED),
    (dict(w_stride=0), abi.E_INVALID), (dict(out_stride=39), abi.E_INVALID), (dict(rows=(1 << 24) + 1), abi.E_INVALID), (dict(n_in=1 << 25, x_stride=1 << 25, w_stride=1 << 25), abi.E_INVALID),
    (dict(rows=1 << 24, n_out=1 << 17, out_stride=1 << 17), abi.E_INVALID), (dict(out=16), abi.E_INVALID), (dict(out=32), abi.E_INVALID)])
def test_products_refuse(change, status):
    refused(rt.dev_linear, LINEAR, change, status)
    refused(rt.dev_gated_linear, GATED, change, status)


def test_each_product_has_its_own_parts():
    refused(rt.dev_linear, LINEAR, dict(up=64, up_stride=64), abi.E_INVALID)
    refused(rt.dev_linear, LINEAR, dict(up_bias=64), abi.E_INVALID)
    refused(rt.dev_linear, LINEAR, dict(residual=64, residual_stride=8), abi.E_INVALID)
    refused(rt.dev_linear, LINEAR, dict(residual=48, residual_stride=48), abi.E_INVALID)
    refused(rt.dev_gated_linear, GATED, dict(residual=64, residual_stride=40), abi.E_INVALID)
    refused(rt.dev_gated_linear, GATED, dict(up_stride=60), abi.E_INVALID)
    refused(rt.dev_gated_linear, GATED, dict(out=64), abi.E_INVALID)
    refused(rt.dev_gated_linear, GATED, dict(up_stride=65), abi.E_UNSUPPORTED)
    for missing in ("x_scale", "w_scale"):
        refused(rt.dev_linear, CODED, {missing: None}, abi.E_INVALID)
    refused(rt.dev_linear, CODED, dict(x_stride=72), abi.E_UNSUPPORTED)
    refused(rt.dev_gated_linear, CODED | dict(up=64, up_stride=64), {}, abi.E_INVALID)
    for call in (rt.dev_linear, rt.dev_gated_linear, rt.dev_norm_rows):
        with pytest.raises(rt.MimirB200Error) as e:
            rt.check(getattr(rt.lib(), "mimir_b200_" + call.__name__)(None, None))
        assert e.value.status == abi.E_INVALID
