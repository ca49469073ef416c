"""Norms of rows at the ends of fp32's range, and of long rows off their boundary."""
import numpy as np
import pytest
import torch

from mimir_framework_b200 import abi
from layer_ref import NORM_UNITS, d, e4m3_half_step, norm_rows, normal, padded
from serving_ref import TORCH, half_step
from test_gpu_layer_calls import call_norm, check_norm

pytestmark = pytest.mark.gpu
F32, F16, BF16, E4M3 = abi.T_F32, abi.T_F16, abi.T_BF16, abi.T_E4M3
STEP = 2.0**-149  # of fp32's smallest numbers


def check_codes(x, gamma, eps, y, scale):
    """Codes and scales of a norm without a residual, where the scale may be one of fp32's smallest numbers.  What the codes are divided by is the scale over
    a factor below two, rounded (half a step); the elements are two products (half a step each) before that."""
    _, v = norm_rows(d(x), None, None if gamma is None else d(gamma), True, eps)
    top = np.abs(v).max(1)
    assert (top > 0).all()
    assert np.all(np.abs(d(scale) - top / 448) <= top / 448 * (NORM_UNITS + 2 * 2.0**-24) + 1.5 * STEP)
    part = (top / 448)[:, None]
    q = v / part
    near = np.abs(q) * (2 * NORM_UNITS + 4 * 2.0**-24 + STEP / part) + 2 * STEP / part
    off, bound = np.abs(d(y) - q), e4m3_half_step(np.abs(q) + near) + near
    assert np.all(off <= bound), (off / bound).max(1)


@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("with_gamma", [False, True])
@pytest.mark.parametrize("n", [40, 300, 1000, 2000, 9000, 20000])
def test_norms_of_small_and_large_rows(backend, n, with_gamma, type_):
    """Rows of one size each.  (What memory holds of an element is exact, however few bits it has; bfloat16 holds zeros of the smallest.)"""
    sizes = [1e-41, 1e-39, 1e-38, 3e-36, 1e-30, 1e-22, 1e-15, 1.0, 1e15, 1e18, 1e25, 5e37]
    x = (normal(len(sizes), n, seed=n).clamp_(-3, 3).double() * torch.tensor(sizes, dtype=torch.float64, device="cuda")[:, None]).to(TORCH[type_])
    some = (x != 0).any(1)
    gamma = 1.0 + normal(n, seed=2, scale=0.3) if with_gamma else None
    for eps in (0.0, 1e-30, 1e-12, 1e-5):
        y, scale = torch.empty(len(sizes), n, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(len(sizes), device="cuda")
        call_norm(backend, x, y, E4M3, type_, gamma=gamma, scale=scale, eps=eps)
        check_codes(x[some], gamma, eps, y.view(torch.uint8)[some].view(torch.float8_e4m3fn), scale[some])
        for y_type in (F32, BF16):
            z = torch.empty(len(sizes), n, dtype=TORCH[y_type], device="cuda")
            call_norm(backend, x, z, y_type, type_, gamma=gamma, eps=eps)
            _, v = norm_rows(d(x[some]), None, None if gamma is None else d(gamma), True, eps)
            # (two products, each half a step off where they are that small, the first one's then times gamma)
            assert np.all(np.abs(d(z[some]) - v) <= np.abs(v) * (half_step(y_type) * 1.001 + NORM_UNITS) + (3 * STEP if y_type == F32 else 2.0**-133))
    backend.check_device()


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("n", [40, 300, 1000, 2000, 9000, 20000])
def test_codes_of_a_norm_whose_row_has_nothing_to_scale_by(backend, n, type_):
    """Zeros, infinities and what is not a number: v by its definition, the scale over what is finite of it."""
    x = normal(8, n, seed=n, dtype=TORCH[type_])
    x[0], x[1] = 0.0, -0.0
    x[2, n // 2] = float("nan")
    x[3, 3] = float("inf")
    x[4, ::2] = -float("inf")
    x[5] = float("nan")
    gamma = 1.0 + normal(n, seed=2, scale=0.3)
    for eps in (1e-5, 0.0):
        y, scale = torch.full((8, n), 5.0, device="cuda").to(torch.float8_e4m3fn), torch.full((8,), 5.0, device="cuda")
        call_norm(backend, x, y, E4M3, type_, gamma=gamma, scale=scale, eps=eps)
        got, s = d(y), d(scale)
        assert (s[:6] == 0).all()  # (nothing finite, or zeros)
        if eps > 0:
            assert (got[:2] == 0).all()
        else:
            assert np.isnan(got[:2]).all()  # 0 / 0
        assert np.isnan(got[2]).all() and np.isnan(got[5]).all()  # (the mean is none)
        # over an infinite mean: 0, and infinity / infinity
        assert np.array_equal(np.isnan(got[3]), np.arange(n) == 3) and (got[3][np.arange(n) != 3] == 0).all()
        assert np.isnan(got[4, ::2]).all() and (got[4, 1::2] == 0).all()
        check_norm(x[6:], None, gamma, True, eps, type_, E4M3, y.view(torch.uint8)[6:].view(torch.float8_e4m3fn), None, scale[6:])
    backend.check_device()


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("y_type", [F32, F16, BF16, E4M3])
@pytest.mark.parametrize("n", [2049, 8193, 9001, 12289, 16383, 16391, 20001, 32761, 32768])
def test_long_rows_off_their_boundary(backend, n, y_type, type_):
    """An odd number of elements from one row to the next: every row starts somewhere else."""
    rows = 9
    x, r = normal(rows, n, seed=n, scale=3.0, dtype=TORCH[type_]), normal(rows, n, seed=n + 1, dtype=TORCH[type_])
    gamma = 1.0 + normal(n + 1, seed=2, scale=0.3)[1:]
    wide = -(-n // 2) * 2
    for lead, residual, norm in ((1, r, True), (3, None, False), (5, None, True)):
        a, b = padded(x, wide + lead, lead=lead), None if residual is None else padded(residual, wide + 3 * lead, lead=lead + 2)
        y = torch.full((rows + 1, wide + 5 * lead), -7.0, device="cuda").to(TORCH[y_type])
        total = torch.full((rows + 1, wide + 7 * lead), -7.0, device="cuda").to(TORCH[type_])
        scale = torch.full((rows + 1,), -7.0, device="cuda") if y_type == E4M3 else None
        g = gamma if norm else None
        call_norm(backend, a, y[:, :n], y_type, type_, residual=b, total=total, gamma=g, scale=scale, norm=norm)
        backend.check_device()
        check_norm(x, residual, g, norm, 1e-5, type_, y_type, y[:rows, :n], total[:rows, :n], None if scale is None else scale[:rows])
        for t in (y, total):
            t = t.float()
            assert (t[:rows, n:] == t[rows, n - 1]).all() and (t[rows] == t[rows, 0]).all()
        assert scale is None or scale[rows] == -7
        if y_type == type_:  # in place: as into memory of its own
            z = padded(x, wide + lead, lead=lead)
            call_norm(backend, z, z, type_, type_, residual=b, gamma=g, norm=norm)
            assert torch.equal(z, y[:rows, :n])
