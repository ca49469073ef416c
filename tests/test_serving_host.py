"""Host side of the serving calls: the rotary plan's steps, struct layouts and the refusals that need no device (CPU)."""
import ctypes
import math
import os
import subprocess
from fractions import Fraction

import pytest

from mimir_framework_b200 import abi, runtime as rt

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = ("MimirRopeSpec", "MimirRopePlan", "MimirPagedCache", "MimirPagedBatch", "MimirPagedAttention")


def test_struct_layouts_match_the_header(tmp_path):
    lines, want = [], []
    for name in STRUCTS:
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


def frequency(i, rot, base=10000.0, scaling="none", factor=1.0, low=1.0, high=1.0, original_len=1.0):
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "bands":
        part = (original_len * f / (2 * math.pi) - low) / (high - low)
        part = min(1.0, max(0.0, part))
        return f * (part + (1 - part) / factor)
    if scaling == "ramp":
        place = [rot * math.log(original_len / (2 * math.pi * r)) / (2 * math.log(base)) for r in (high, low)]
        a, b = max(math.floor(place[0]), 0), min(math.ceil(place[1]), rot - 1)
        w = min(1.0, max(0.0, (i - a) / (b - a if b > a else 0.001)))
        return f * ((1 - w) + w / factor)
    return f


@pytest.mark.parametrize("spec", [
    dict(rot_dim=64), dict(rot_dim=2, base=500000.0), dict(rot_dim=256, interleaved=True), dict(rot_dim=128, scaling="linear", factor=4.0),
    dict(rot_dim=128, base=500000.0, scaling="bands", factor=8.0, low=1.0, high=4.0, original_len=8192.0),
    dict(rot_dim=96, scaling="ramp", factor=16.0, low=1.0, high=32.0, original_len=4096.0, magnitude=1.25)])
def test_rope_plan_holds_each_frequency_as_a_part_of_a_turn(spec):
    plan = rt.rope_plan(**spec)
    back = rt.rope_plan(**spec, inverse=True)
    rot = spec["rot_dim"]
    assert plan.rot_dim == rot and plan.interleaved == int(spec.get("interleaved", False)) and plan.magnitude == spec.get("magnitude", 1.0)
    names = ("base", "scaling", "factor", "low", "high", "original_len")
    for i in range(rot // 2):
        turns = frequency(i, rot, **{n: spec[n] for n in names if n in spec}) / (2 * math.pi)
        # Python's value has some ten roundings of 2^-53; the plan's own is below that
        assert abs(float(Fraction(plan.step[i], 1 << 64)) - turns) <= 16 * 2.0**-53 * turns + 2.0**-64
        assert (plan.step[i] + back.step[i]) % (1 << 64) == 0
    assert all(plan.step[i] == 0 for i in range(rot // 2, abi.MAX_ROPE_PAIRS))


@pytest.mark.parametrize("spec", [
    dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258), dict(rot_dim=64, base=1.0), dict(rot_dim=64, base=float("inf")), dict(rot_dim=64, base=float("nan")),
    dict(rot_dim=64, scaling="linear"), dict(rot_dim=64, scaling="linear", factor=-2.0), dict(rot_dim=64, scaling="bands", factor=2.0, low=4.0, high=1.0, original_len=100.0),
    dict(rot_dim=64, scaling="ramp", factor=2.0, low=1.0, high=4.0), dict(rot_dim=64, magnitude=-1.0), dict(rot_dim=64, magnitude=float("nan"))])
def test_rope_plan_refuses(spec):
    with pytest.raises(rt.MimirB200Error) as e:
        rt.rope_plan(**spec)
    assert e.value.status == abi.E_INVALID


def test_division_by_the_page_size_is_exact():
    """The kernels divide a key by the page size as (umulhi(m, n) + n) >> l."""
    for d in [1, 2, 7, 8, 16, 24, 40, 56, 64, 120, 128, 1000, 4096, 65536, (1 << 30) + 8]:
        l = (d - 1).bit_length()
        m = (((1 << l) - d) << 32) // d + 1
        assert m < 1 << 32
        for n in {0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, 12345678, (1 << 31) - 1, (1 << 31) - d, ((1 << 31) - 1) // d * d, ((1 << 31) - 1) // d * d - 1}:
            if 0 <= n < 1 << 31:
                q = (m * n >> 32) + n
                assert q < 1 << 32 and q >> l == n // d, (n, d)


def call(**change):
    """A refused call changes one number of a set that passes the checks of sizes."""
    c = dict(k=16, v=16, type=abi.T_F16, n_pages=4, page_size=16, kv_heads=2, head_dim=64, page_stride=2048, slot_stride=128, head_stride=64)
    b = dict(row_start=16, kv_len=16, page_table=16, table_stride=4, n_seqs=1, n_rows=1, max_rows=1, max_kv=64)
    a = dict(q=16, out=16, type=abi.T_F16, heads=4, row_stride=256, head_stride=64, out_row_stride=256, out_head_stride=64, scale=0.125)
    for k, v in change.items():
        part, name = k.split("_", 1)
        {"c": c, "b": b, "a": a}[part][name] = v
    return rt.paged_cache(**c), rt.paged_batch(**b), rt.paged_attention(**a)


CACHE_REFUSED = [("c_type", 5, abi.E_INVALID), ("c_type", -1, abi.E_INVALID), ("c_n_pages", 0, abi.E_INVALID), ("c_kv_heads", 0, abi.E_INVALID),
                 ("c_page_size", 0, abi.E_INVALID), ("c_page_size", 12, abi.E_UNSUPPORTED), ("c_head_dim", 20, abi.E_UNSUPPORTED),
                 ("c_head_dim", 264, abi.E_UNSUPPORTED), ("c_head_dim", -8, abi.E_INVALID), ("c_slot_stride", 100, abi.E_UNSUPPORTED),
                 ("c_page_stride", -8, abi.E_UNSUPPORTED), ("b_n_seqs", -1, abi.E_INVALID), ("b_n_rows", -1, abi.E_INVALID), ("b_max_kv", -1, abi.E_INVALID),
                 ("b_table_stride", -1, abi.E_INVALID)]
ATTENTION_REFUSED = [("a_type", abi.T_I8, abi.E_INVALID), ("a_heads", 3, abi.E_INVALID), ("a_heads", 0, abi.E_INVALID), ("a_window", -1, abi.E_INVALID),
                     ("a_scale", float("nan"), abi.E_INVALID), ("a_row_stride", 12, abi.E_UNSUPPORTED), ("a_out_head_stride", -8, abi.E_UNSUPPORTED),
                     ("c_type", abi.T_F32, abi.E_UNSUPPORTED), ("c_type", abi.T_BF16, abi.E_UNSUPPORTED)]


@pytest.mark.parametrize("name,value,status", CACHE_REFUSED)
def test_cache_calls_refuse_sizes(name, value, status):
    cache, batch, att = call(**{name: value})
    for f in (lambda: rt.dev_cache_write(cache, batch, 16, 16, abi.T_F16, 128, 64), lambda: rt.dev_cache_read(cache, batch, 16, 1, 16, 16, abi.T_F16, 128, 64),
              lambda: rt.dev_paged_attention(cache, batch, att), lambda: rt.paged_attention_workspace(cache, batch, att)):
        with pytest.raises(rt.MimirB200Error) as e:
            f()
        assert e.value.status == status


@pytest.mark.parametrize("name,value,status", ATTENTION_REFUSED)
def test_attention_refuses(name, value, status):
    cache, batch, att = call(**{name: value})
    for f in (lambda: rt.dev_paged_attention(cache, batch, att), lambda: rt.paged_attention_workspace(cache, batch, att)):
        with pytest.raises(rt.MimirB200Error) as e:
            f()
        assert e.value.status == status


@pytest.mark.parametrize("name,value", [("c_slot_stride", 0), ("c_head_stride", 0), ("c_page_stride", 0), ("c_page_stride", 1 << 38), ("c_slot_stride", 1 << 38)])
def test_cache_strides_that_fold_or_run_away_are_refused(name, value):
    test_cache_calls_refuse_sizes(name, value, abi.E_UNSUPPORTED)


def test_more_rows_and_heads_than_32_bits_are_refused():
    cache, batch, att = call(b_n_rows=1 << 29, b_max_rows=1 << 29, a_heads=4)
    for f in (lambda: rt.dev_paged_attention(cache, batch, att), lambda: rt.paged_attention_workspace(cache, batch, att)):
        with pytest.raises(rt.MimirB200Error, match="too many rows") as e:
            f()
        assert e.value.status == abi.E_INVALID


def test_row_types_and_sizes_are_refused():
    cache, batch, _ = call()
    plan = rt.rope_plan(64)
    for f in (lambda: rt.dev_cache_write(cache, batch, 16, 16, abi.T_I8, 128, 64), lambda: rt.dev_cache_read(cache, batch, 16, -1, 16, 16, abi.T_F16, 128, 64),
              lambda: rt.dev_rope(plan, 16, 16, 32, 1, 2, 32, (64, 32), (64, 32), abi.T_F32),       # 64 turned of 32
              lambda: rt.dev_rope(plan, 16, 16, 16, 1, 2, 64, (128, 64), (256, 64), abi.T_F32),     # in place, other strides
              lambda: rt.dev_rope(plan, 16, 16, 32, -1, 2, 64, (128, 64), (128, 64), abi.T_F32),
              lambda: rt.dev_rope(plan, 16, 16, 32, 1, 2, 64, (-128, 64), (128, 64), abi.T_F32),
              lambda: rt.dev_rope(plan, 16, 16, 32, 1, 2, 64, (128, 64), (128, 64), abi.T_E4M3),
              lambda: rt.dev_rope(abi.MimirRopePlan(), 16, 16, 32, 1, 2, 64, (128, 64), (128, 64), abi.T_F32),
              lambda: rt.dev_sample_rows(16, abi.T_I8, 1, 10, 10, None, None, None, None, 16, 16),
              lambda: rt.dev_sample_rows(16, abi.T_F32, 1, 0, 10, None, None, None, None, 16, 16),
              lambda: rt.dev_sample_rows(16, abi.T_F32, -1, 10, 10, None, None, None, None, 16, 16),
              lambda: rt.dev_sample_rows(16, abi.T_F32, 1, 10, -10, None, None, None, None, 16, 16),
              lambda: rt.dev_sample_rows(16, abi.T_F32, 1, (1 << 24) + 1, 1 << 25, None, None, None, None, 16, 16)):
        with pytest.raises(rt.MimirB200Error) as e:
            f()
        assert e.value.status == abi.E_INVALID
