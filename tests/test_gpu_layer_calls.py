"""A layer's norms and products on the GPU against their definitions in 64 bits, and a layer of them together with the serving calls."""
import math

import numpy as np
import pytest
import torch

from mimir_framework_b200 import abi
from layer_ref import ACTS, NORM_UNITS, Operand, act, act_off, check_product, d, e4m3_half_step, linear_args, norm_rows, normal, padded, product, rounded
from serving_ref import TORCH, Pages, half_step, sample

pytestmark = pytest.mark.gpu
F32, F16, BF16, I8, E4M3 = abi.T_F32, abi.T_F16, abi.T_BF16, abi.T_I8, abi.T_E4M3


# ---- norms --------------------------------------------------------------------------------------------------------------------------
def call_norm(backend, x, y, y_type, type_, residual=None, total=None, gamma=None, scale=None, norm=True, eps=1e-5, stream=0, rows=None):
    a = backend.norm_rows(x.data_ptr(), y.data_ptr(), x.shape[0] if rows is None else rows, x.shape[1], type_, y_type, x.stride(0), y.stride(0),
                          None if gamma is None else gamma.data_ptr(), None if residual is None else residual.data_ptr(),
                          0 if residual is None else residual.stride(0), None if total is None else total.data_ptr(),
                          0 if total is None else total.stride(0), None if scale is None else scale.data_ptr(), norm, eps)
    backend.dev_norm_rows(a, stream)
    torch.cuda.synchronize()


def check_norm(x, residual, gamma, norm, eps, type_, y_type, y, total, scale):
    s, v = norm_rows(d(x), None if residual is None else d(residual), None if gamma is None else d(gamma), norm, eps)
    if total is not None:
        assert np.all(np.abs(d(total) - s) <= np.abs(s) * (half_step(type_) + 2.0**-23) + (2.0**-25 if type_ == F16 else 0))
    units = NORM_UNITS if norm else 2.0**-24
    if y_type != E4M3:
        assert np.all(np.abs(d(y) - v) <= np.abs(v) * (half_step(y_type) * 1.001 + units) + (2.0**-25 if y_type == F16 else 1e-40))
        return
    top = np.abs(v).max(1)
    assert np.all(np.abs(d(scale) - top / 448) <= top / 448 * (units + 2 * 2.0**-24) + 1e-44)
    q = v / np.where(top > 0, top / 448, 1)[:, None]
    # the quotient's own errors: v's, the scale's, the division's
    near = np.abs(q) * (2 * units + 4 * 2.0**-24)
    assert np.all(np.abs(d(y) - q) <= e4m3_half_step(np.abs(q) + near) + near)


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("y_type", [F32, F16, BF16, E4M3])
@pytest.mark.parametrize("rows,n", [(1, 1), (5, 3), (3, 256), (9, 257), (2, 500), (6, 1024), (3, 1025), (4, 4096), (2, 5003), (1, 16384), (2, 32761), (2, 32768)])
def test_norm_rows(backend, rows, n, y_type, type_):
    x, r = normal(rows, n, seed=n, scale=3.0, dtype=TORCH[type_]), normal(rows, n, seed=n + 1, dtype=TORCH[type_])
    gamma = 1.0 + normal(n, seed=2, scale=0.3)
    wide = -(-n // 16) * 16
    for lead in (0, 1) if n < 2000 else (0,):  # (rows on 16 bytes and off them)
        for residual, norm in ((r, True), (None, True), (r, False), (None, False)):
            a, b = padded(x, wide + lead, lead=lead), None if residual is None else padded(residual, wide + 3 * lead, lead=lead)
            y = torch.full((rows + 1, wide + 5 * lead), -7.0, device="cuda").to(TORCH[y_type])
            total = torch.full((rows + 1, wide + 7 * lead), -7.0, device="cuda").to(TORCH[type_])
            scale = torch.full((rows + 1,), -7.0, device="cuda") if y_type == E4M3 else None
            g = gamma if norm and residual is not None else None
            a_args = dict(residual=b, total=total, gamma=g, scale=scale, norm=norm)
            call_norm(backend, a, y[:, :n], y_type, type_, **a_args)
            backend.check_device()
            check_norm(x, residual, g, norm, 1e-5, type_, y_type, y[:rows, :n], total[:rows, :n], None if scale is None else scale[:rows])
            for t in (y, total):
                t = t.float()
                assert (t[:rows, n:] == t[rows, n - 1]).all() and (t[rows] == t[rows, 0]).all()
            assert scale is None or scale[rows] == -7


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("y_type", [F32, BF16, E4M3])
@pytest.mark.parametrize("rows,n", [(593, 8200), (2000, 12288), (1200, 16384)])
def test_norm_of_many_long_rows(backend, rows, n, y_type, type_):
    """More rows than the device holds at once: every CTA has several, the last of them fewer."""
    x = normal(rows, n, seed=rows, scale=2.0, dtype=TORCH[type_])
    x[rows // 2, 5] = float("nan")
    for norm in (True, False):
        y, scale = torch.full((rows + 1, n + 16), -7.0, device="cuda").to(TORCH[y_type]), torch.full((rows + 1,), -7.0, device="cuda")
        call_norm(backend, x, y[:, :n], y_type, type_, scale=scale if y_type == E4M3 else None, norm=norm, rows=rows)
        backend.check_device()
        fine = [0, 1, rows // 2 - 1, rows // 2 + 1, rows - 2, rows - 1] + list(range(3, rows, 97))
        part = y[:, :n].view(torch.uint8 if y_type == E4M3 else y.dtype)[fine].view(TORCH[y_type])
        check_norm(x[fine], None, None, norm, 1e-5, type_, y_type, part, None, scale[fine])
        rest = y.float()
        assert rest[rows // 2, 5].isnan() and rest[rows // 2, :n].isnan().all() == norm
        assert (rest[:, n:] == rest[rows, 0]).all() and (rest[rows] == rest[rows, 0]).all() and scale[rows] == -7
        same = torch.empty_like(x)
        if y_type == type_:
            call_norm(backend, x.clone(), same, type_, type_, norm=norm)
            z = x.clone()
            call_norm(backend, z, z, type_, type_, norm=norm)
            assert torch.equal(z.nan_to_num(3.0), same.nan_to_num(3.0))


@pytest.mark.parametrize("type_", [F32, BF16])
def test_norm_rows_in_place(backend, type_):
    x, r = normal(7, 768, seed=1, dtype=TORCH[type_]), normal(7, 768, seed=2, dtype=TORCH[type_])
    want_y, want_s = torch.empty_like(x), torch.empty_like(x)
    call_norm(backend, x, want_y, type_, type_, residual=r, total=want_s)
    for total, y in (("x", "r"), ("r", "x"), ("r", None), (None, "x")):
        a, b = x.clone(), r.clone()
        of = {"x": a, "r": b, None: torch.empty_like(x)}
        s = of[total] if total else None
        call_norm(backend, a, of[y], type_, type_, residual=b, total=s)
        assert torch.equal(of[y], want_y) and (s is None or torch.equal(s, want_s))


def test_norm_rows_zeros_and_numbers_that_are_none(backend):
    """A row's infinities and what is not a number stay in it; zeros, the smallest numbers and the largest."""
    for n in (40, 300, 2000, 9000):
        x = normal(9, n, seed=n)
        x[1] = 0.0
        x[2, n // 2] = float("nan")
        x[3, 3] = float("inf")
        x[4, ::2] = -float("inf")
        x[5] *= 1e-42
        x[6] *= 1e18
        x[7, :] = -0.0
        fine = [0, 1, 5, 6, 7, 8]
        y, scale = torch.empty(9, n, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(9, device="cuda")
        call_norm(backend, x, y, E4M3, F32, scale=scale, norm=False)
        got, xd = d(y), d(x)
        check_norm(x[[0, 6, 8]], None, None, False, 0, F32, E4M3, y.view(torch.uint8)[[0, 6, 8]].view(torch.float8_e4m3fn), None, scale[[0, 6, 8]])
        assert (got[[1, 7]] == 0).all() and (d(scale)[[1, 7]] == 0).all()
        assert np.isnan(got[2]).sum() == 1 and np.isnan(got[2, n // 2]) and got[3, 3] == 448 and (got[4, ::2] == -448).all()
        others = np.arange(n) != 3
        top = np.abs(xd[3, others]).max()
        assert abs(d(scale)[3] - top / 448) <= top / 448 * 2.0**-22
        # (of the smallest a scale is a whole number of fp32's smallest step, and as far off as that makes it)
        assert np.isfinite(got[5]).all() and np.abs(got[5]).max() <= 448
        z = torch.empty_like(x)
        call_norm(backend, x, z, F32, F32, eps=1e-6)
        check_norm(x[[0, 8]], None, None, True, 1e-6, F32, F32, z[[0, 8]], None, None)
        assert (z[1] == 0).all() and (z[7] == 0).all() and z[2].isnan().all() and z[3, 3].isnan() and (d(z)[3, others] == 0).all()
        assert np.allclose(d(z)[6], d(x)[6] / np.sqrt((d(x)[6] ** 2).mean()), rtol=1e-5)
    backend.check_device()


# ---- products -------------------------------------------------------------------------------------------------------------------------
ROWS = [1, 2, 16, 17, 40, 64, 65, 129, 200, 257, 520]


@pytest.mark.parametrize("type_,out_type", [(F16, F16), (BF16, BF16), (E4M3, BF16), (BF16, F32), (E4M3, F32), (F16, BF16), (E4M3, F16)])
@pytest.mark.parametrize("rows", ROWS)
def test_linear(backend, rows, type_, out_type):
    for i, (n_in, n_out) in enumerate([(64, 128), (1, 1), (100, 130), (1000, 300), (513, 33), (4096, 256)]):
        check_product(backend, rows, n_in, n_out, type_, out_type, name=list(ACTS)[(rows + i) % 6], bias=i % 2 == 0, residual=i % 3 != 0, seed=rows + i)


@pytest.mark.parametrize("type_,out_type", [(F16, F16), (BF16, BF16), (E4M3, BF16), (BF16, F32), (E4M3, F32)])
@pytest.mark.parametrize("rows", ROWS)
def test_gated_linear(backend, rows, type_, out_type):
    for i, (n_in, n_out) in enumerate([(64, 128), (3, 1), (100, 130), (1000, 301), (4096, 64)]):
        check_product(backend, rows, n_in, n_out, type_, out_type, name=list(ACTS)[(rows + i) % 6], bias=i % 2 == 0, gated=True, seed=rows + i)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,n_in,n_out,type_,out_type", [
    (3000, 512, 1111, BF16, BF16), (1500, 2000, 2049, E4M3, F16), (4100, 128, 700, F16, F32), (2048, 4096, 1024, E4M3, F32), (300, 12288, 512, BF16, BF16),
    (1, 16384, 5000, E4M3, F32), (48, 9000, 4096, F16, F16), (128, 64, 20000, BF16, F32), (7, 40, 32000, E4M3, BF16)])
def test_products_of_larger_sizes(backend, rows, n_in, n_out, type_, out_type, gated):
    check_product(backend, rows, n_in, n_out, type_, out_type, name="silu", residual=not gated, gated=gated, seed=3, out_wide=-(-n_out // 16) * 16)


@pytest.mark.parametrize("rows", [3, 70, 600, 2500])
@pytest.mark.parametrize("out_type", [F32, F16, BF16])
def test_results_of_every_alignment(backend, rows, out_type):
    """Rows of the result on 32 bytes, on 16, on their elements' size only."""
    for out_wide, lead in [(320, 0), (320, 8), (304, 4), (301, 0), (305, 1)]:
        check_product(backend, rows, 96, 299, BF16, out_type, residual=True, seed=lead, out_wide=out_wide, lead=lead)
        check_product(backend, rows, 96, 299, E4M3, out_type, name="gelu", gated=True, seed=lead, out_wide=out_wide, lead=lead)


@pytest.mark.parametrize("rows", [1, 33, 300, 1100])
def test_residual_in_place(backend, rows):
    for type_, out_type in ((BF16, BF16), (E4M3, F32)):
        a = check_product(backend, rows, 520, 384, type_, out_type, name="silu", residual=True, seed=5)
        b = check_product(backend, rows, 520, 384, type_, out_type, name="silu", residual=True, seed=5, in_place=True)
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 30, 300, 1400])
@pytest.mark.parametrize("type_", [F16, E4M3])
def test_numbers_that_are_none_stay_in_their_row_and_feature(backend, rows, type_):
    n_in, n_out = 200, 270
    x, w, u = Operand(rows, n_in, type_, 1), Operand(n_out, n_in, type_, 2, 0.1), Operand(n_out, n_in, type_, 3, 0.1)
    out = torch.empty(rows, n_out, device="cuda")
    a = linear_args(x, w, out, type_, F32, rows, n_in, n_out)
    g = linear_args(x, w, out, type_, F32, rows, n_in, n_out, up=u.at(), up_stride=u.stride, up_scale=u.scale_at(), activation=abi.ELT_SILU)
    calls = [lambda: backend.dev_linear(a), lambda: backend.dev_gated_linear(g)]
    clean = []
    for f in calls:
        f()
        clean.append(d(out))
    x.x[rows // 2, 17] = float("nan")
    w.x[5, 3] = float("nan")
    w.x[n_out - 1, n_in - 1] = float("nan")
    for f, want in zip(calls, clean):
        f()
        got = d(out)
        bad = np.zeros((rows, n_out), bool)
        bad[rows // 2], bad[:, [5, n_out - 1]] = True, True
        assert np.array_equal(np.isnan(got), bad) and np.array_equal(got[~bad], want[~bad])
    backend.check_device()


@pytest.mark.parametrize("rows", [1, 64, 700])
def test_the_same_call_gives_the_same_bits_and_rows_do_not_depend_on_each_other(backend, rows):
    x, w = Operand(rows, 1000, BF16, 1), Operand(500, 1000, BF16, 2)
    first = None
    for _ in range(5):
        out = torch.empty(rows, 500, device="cuda")
        backend.dev_linear(linear_args(x, w, out, BF16, F32, rows, 1000, 500))
        torch.cuda.synchronize()
        first = out if first is None else first
        assert torch.equal(out, first)


def test_results_beyond_32_bits_of_offset(backend):
    """Rows of the result and of an operand more than 2^32 bytes apart."""
    wide, rows = (1 << 31) + 64, 3
    big = torch.zeros(rows, wide, dtype=torch.bfloat16, device="cuda")
    x = normal(rows, 128, seed=1, dtype=torch.bfloat16)
    big[:, :128] = x
    w = Operand(72, 128, BF16, 2)
    out = big[:, 256 : 256 + 72]
    a = backend.linear(big.data_ptr(), w.at(), out.data_ptr(), rows, 128, 72, BF16, BF16, wide, w.stride, wide)
    backend.dev_linear(a)
    want = torch.empty(rows, 72, dtype=torch.bfloat16, device="cuda")
    backend.dev_linear(backend.linear(x.data_ptr(), w.at(), want.data_ptr(), rows, 128, 72, BF16, BF16, 128, w.stride, 72))
    n = backend.norm_rows(big.data_ptr(), big[:, 512:].data_ptr(), rows, 128, BF16, BF16, wide, wide)
    backend.dev_norm_rows(n)
    torch.cuda.synchronize()
    backend.check_device()
    assert torch.equal(out, want)
    check_norm(x, None, None, True, 1e-5, BF16, BF16, big[:, 512 : 512 + 128], None, None)


# ---- refusals that need a device ----------------------------------------------------------------------------------------------------------
def test_pointers_are_looked_at(backend):
    x, w, y = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda"), torch.full((4, 8), -7.0, device="cuda")
    host = torch.zeros(4, 64, dtype=torch.bfloat16)
    good = dict(x=x.data_ptr(), w=w.data_ptr(), out=y.data_ptr(), rows=4, n_in=64, n_out=8, type=BF16, out_type=F32, x_stride=64, w_stride=64, out_stride=8)
    norm = dict(x=x.data_ptr(), y=w.data_ptr(), rows=4, n=64, type=BF16, y_type=BF16, x_stride=64, y_stride=64)
    E_INVALID, E_UNSUPPORTED = abi.E_INVALID, abi.E_UNSUPPORTED
    for change, status in [(dict(x=None), E_INVALID), (dict(w=host.data_ptr()), E_INVALID), (dict(out=None), E_INVALID), (dict(x=x.data_ptr() + 8), E_UNSUPPORTED),
                           (dict(out=y.data_ptr() + 2), E_INVALID), (dict(bias=host.data_ptr()), E_INVALID), (dict(bias=y.data_ptr() + 2), E_INVALID),
                           (dict(residual=y.data_ptr() + 1, residual_stride=8), E_INVALID)]:
        with pytest.raises(backend.MimirB200Error) as e:
            backend.dev_linear(backend.linear(**(good | change)))
        assert e.value.status == status, change
    with pytest.raises(backend.MimirB200Error) as e:
        backend.dev_gated_linear(backend.linear(**good))
    assert e.value.status == E_INVALID
    for change, status in [(dict(x=None), E_INVALID), (dict(y=host.data_ptr()), E_INVALID), (dict(x=x.data_ptr() + 1), E_INVALID), (dict(gamma=host.data_ptr()), E_INVALID)]:
        with pytest.raises(backend.MimirB200Error) as e:
            backend.dev_norm_rows(backend.norm_rows(**(norm | change)))
        assert e.value.status == status, change
    torch.cuda.synchronize()
    assert (y == -7).all()
    # no rows: nothing is looked at
    backend.dev_linear(backend.linear(**(good | dict(rows=0, x=None, out=None))))
    backend.dev_norm_rows(backend.norm_rows(**(norm | dict(rows=0, x=None))))


# ---- sizes between the two kernels, and every division of the inputs -----------------------------------------------------------------------
@pytest.mark.parametrize("type_,out_type", [(BF16, F32), (E4M3, F32), (F16, F16), (E4M3, BF16)])
@pytest.mark.parametrize("rows,n_in,n_out", [(700, 8, 3000), (1111, 129, 1500), (2049, 257, 513), (900, 5000, 1300), (5000, 64, 40), (770, 1024, 4096), (258, 3000, 4096), (130, 8192, 130)])
@pytest.mark.parametrize("gated", [False, True])
def test_products_of_many_shapes(backend, rows, n_in, n_out, type_, out_type, gated):
    check_product(backend, rows, n_in, n_out, type_, out_type, name="gelu" if gated else "none", residual=not gated, gated=gated, seed=rows)


@pytest.mark.parametrize("type_", [BF16, E4M3])
@pytest.mark.parametrize("n_in", [512, 1000, 2048, 4096, 8000, 20000])
@pytest.mark.parametrize("n_out", [8, 100, 520, 4096])
def test_products_of_few_rows_whose_inputs_are_shared_out(backend, n_in, n_out, type_):
    """From one CTA for all of n_in to eight of them, with as many rows as make one unit or several."""
    for rows in (1, 16, 48, 100, 160):
        check_product(backend, rows, n_in, n_out, type_, F32 if rows % 3 else BF16, residual=rows > 16, seed=rows + n_in)
        if n_out < 4096:
            check_product(backend, rows, n_in, n_out, type_, BF16, name="silu", gated=True, seed=rows + n_in)


def test_weights_beyond_32_bits_of_offset(backend):
    stride, n_out, n_in = 1 << 27, 18, 200
    big = torch.empty(n_out, stride, dtype=torch.bfloat16, device="cuda")
    w = normal(n_out, n_in, seed=1, dtype=torch.bfloat16)
    big[:, :n_in] = w
    for rows in (3, 1500):
        x = normal(rows, n_in, seed=2, dtype=torch.bfloat16)
        got, want = torch.empty(rows, n_out, device="cuda"), torch.empty(rows, n_out, device="cuda")
        backend.dev_linear(backend.linear(x.data_ptr(), big.data_ptr(), got.data_ptr(), rows, n_in, n_out, BF16, F32, n_in, stride, n_out))
        backend.dev_linear(backend.linear(x.data_ptr(), w.data_ptr(), want.data_ptr(), rows, n_in, n_out, BF16, F32, n_in, n_in, n_out))
        torch.cuda.synchronize()
        backend.check_device()
        assert torch.equal(got, want)


# ---- streams and graphs ----------------------------------------------------------------------------------------------------------------------
def test_calls_of_several_streams_at_once(backend):
    """Clusters that share inputs, single CTAs, pairs and norms beside one another: the results are those of one call after the other."""
    sizes = [(40, 4096, 1024, BF16), (1500, 1024, 1536, F16), (3, 2048, 20000, E4M3), (300, 4096, 2048, E4M3)]
    jobs = []
    for i, (rows, n_in, n_out, type_) in enumerate(sizes):
        x, w, u = Operand(rows, n_in, type_, i), Operand(n_out, n_in, type_, i + 10, 0.02), Operand(n_out, n_in, type_, i + 20, 0.02)
        out = torch.empty(2, rows, n_out, device="cuda", dtype=torch.bfloat16)
        a = linear_args(x, w, out[0], type_, BF16, rows, n_in, n_out)
        g = linear_args(x, w, out[1], type_, BF16, rows, n_in, n_out, up=u.at(), up_stride=u.stride, up_scale=u.scale_at(), activation=abi.ELT_SILU)
        y, scale = torch.empty(rows, n_out, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(rows, device="cuda")
        norm = backend.norm_rows(out[0].data_ptr(), y.data_ptr(), rows, n_out, BF16, E4M3, n_out, n_out, y_scale=scale.data_ptr())
        jobs.append((a, g, norm, out, y, scale, (x, w, u)))

    def run(job, stream):
        backend.dev_linear(job[0], stream)
        backend.dev_norm_rows(job[2], stream)
        backend.dev_gated_linear(job[1], stream)

    for job in jobs:
        run(job, 0)
    torch.cuda.synchronize()
    want = [(job[3].clone(), job[4].view(torch.uint8).clone(), job[5].clone()) for job in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(20):
        for job, s in zip(jobs, streams):
            run(job, s.cuda_stream)
    torch.cuda.synchronize()
    backend.check_device()
    for job, (o, y, s) in zip(jobs, want):
        assert torch.equal(job[3], o) and torch.equal(job[4].view(torch.uint8), y) and torch.equal(job[5], s)
    # two graphs at once, on new inputs in the old buffers
    graphs = []
    for job, s in zip(jobs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run(job, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for job in jobs:
        job[3].zero_(), job[5].zero_()
        x = job[6][0].x
        x.copy_(x.flip(0))
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    backend.check_device()
    for job, (o, y, s) in zip(jobs, want):
        x = job[6][0]
        if x.scale is None:  # (8-bit rows keep their scales' places)
            assert torch.equal(job[3], o.flip(1)) and torch.equal(job[5], s.flip(0))


# ---- together -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("coded", [False, True])
def test_a_layer_and_its_tokens(backend, coded):
    """A layer of a small model as it serves: norm, projection, rotary positions, cache, attention, projection with the residual, norm with the
    residual's sum, gated block, logits, a token; a prompt's chunk and then single tokens, the steps captured once and replayed.  Each call is held against
    its definition over what it then read."""
    heads, kv_heads, dim, page, vocab, width, hidden = 6, 2, 64, 16, 301, 384, 1000
    prompt, steps, type_ = [20, 5, 33], 3, BF16
    bf = torch.bfloat16
    p = Pages(prompt, [n + steps for n in prompt], kv_heads, dim, page, F16 if coded else BF16, seed=3)
    wide = (heads + 2 * kv_heads) * dim
    embed = normal(vocab, width, seed=1, dtype=bf)
    op = E4M3 if coded else BF16
    weights = {name: Operand(o, i, op, 20 + k, 1 / math.sqrt(i)) for k, (name, i, o) in enumerate(
        [("qkv", width, wide), ("out", heads * dim, width), ("gate", width, hidden), ("up", width, hidden), ("down", hidden, width), ("head", width, vocab)])}
    gamma = [1.0 + normal(width, seed=40 + i, scale=0.1) for i in range(3)]
    plan = backend.rope_plan(dim, base=500000.0)
    stream = torch.cuda.Stream()

    def buffers(rows):
        n = sum(rows)
        b = {"rows": torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda"), "kv": torch.zeros(3, dtype=torch.int32, device="cuda"),
             "pos": torch.zeros(n, dtype=torch.int32, device="cuda"), "tok": torch.zeros(n, dtype=torch.int64, device="cuda"), "u": torch.zeros(3, device="cuda"),
             "last": torch.zeros(3, dtype=torch.int64, device="cuda"), "ids": torch.zeros(3, dtype=torch.int32, device="cuda"), "logits": torch.zeros(3, vocab, device="cuda")}
        for name, size in (("x", width), ("qkv", wide), ("turned", wide), ("att", heads * dim), ("mid", width), ("sum", width), ("h", hidden), ("end", width)):
            b[name] = torch.zeros(n, size, dtype=bf, device="cuda")
        b["tail"] = torch.zeros(3, width, dtype=bf, device="cuda")
        for name, rows_of, size in (("n1", n, width), ("n2", n, width), ("n3", 3, width), ("a8", n, heads * dim), ("h8", n, hidden)):
            # (rows of 8-bit operands start on 16 bytes)
            b[name] = torch.zeros(rows_of, -(-size // 16) * 16, dtype=TORCH[op], device="cuda")[:, :size]
            b[name + "s"] = torch.zeros(rows_of, device="cuda")
        return b

    def norm(b, x, y, gamma_, s, residual=None, total=None, norm=True):
        backend.dev_norm_rows(backend.norm_rows(
            b[x].data_ptr(), b[y].data_ptr(), b[x].shape[0], b[x].shape[1], type_, op, b[x].stride(0), b[y].stride(0), None if gamma_ is None else gamma_.data_ptr(),
            None if residual is None else b[residual].data_ptr(), width, None if total is None else b[total].data_ptr(), width,
            b[y + "s"].data_ptr() if coded else None, norm), s)

    def operand(b, name):
        class X:
            x, stride, scale = b[name], b[name].stride(0), b[name + "s"] if coded else None
            value = property(lambda self: d(self.x) if self.scale is None else d(self.x) * d(self.scale)[:, None])
            def at(self): return self.x.data_ptr()
            def scale_at(self): return None if self.scale is None else self.scale.data_ptr()
        return X()

    def linear(b, x, w, y, s, residual=None, gated=False, out_type=BF16):
        o, i, ww = b[y].shape[1], weights[w].x.shape[1], weights[w]
        more = {}
        if residual:
            more = dict(residual=b[residual].data_ptr(), residual_stride=b[residual].stride(0))
        if gated:
            up = weights["up"]
            more = dict(up=up.at(), up_stride=up.stride, up_scale=up.scale_at(), activation=abi.ELT_SILU)
        a = linear_args(operand(b, x), ww, b[y], op, out_type, b[x].shape[0], i, o, **more)
        (backend.dev_gated_linear if gated else backend.dev_linear)(a, s)

    def step(b, rows):
        s = torch.cuda.current_stream().cuda_stream
        batch = backend.paged_batch(b["rows"].data_ptr(), b["kv"].data_ptr(), p.dev[2].data_ptr(), p.width, 3, sum(rows), max(rows), 64)
        torch.index_select(embed, 0, b["tok"], out=b["x"])
        norm(b, "x", "n1", gamma[0], s)
        linear(b, "n1", "qkv", "qkv", s)
        b["turned"].copy_(b["qkv"])
        q = b["turned"]
        backend.dev_rope(plan, b["pos"].data_ptr(), q.data_ptr(), q.data_ptr(), sum(rows), heads + kv_heads, dim, (wide, dim), (wide, dim), type_, s)
        backend.dev_cache_write(p.cache(), batch, q[:, heads * dim :].data_ptr(), q[:, (heads + kv_heads) * dim :].data_ptr(), type_, wide, dim, s)
        a = backend.paged_attention(q.data_ptr(), b["att"].data_ptr(), type_, heads, wide, dim, heads * dim, dim, dim**-0.5)
        assert backend.paged_attention_workspace(p.cache(), batch, a) == 0
        backend.dev_paged_attention(p.cache(), batch, a, s)
        norm(b, "att", "a8", None, s, norm=False)
        linear(b, "a8", "out", "mid", s, residual="x")
        norm(b, "mid", "n2", gamma[1], s, residual="x", total="sum")
        linear(b, "n2", "gate", "h", s, gated=True)
        norm(b, "h", "h8", None, s, norm=False)
        linear(b, "h8", "down", "end", s, residual="sum")
        torch.index_select(b["end"], 0, b["last"], out=b["tail"])
        norm(b, "tail", "n3", gamma[2], s)
        linear(b, "n3", "head", "logits", s, out_type=F32)
        backend.dev_sample_rows(b["logits"].data_ptr(), F32, 3, vocab, vocab, None, None, None, None, b["u"].data_ptr(), b["ids"].data_ptr(), None, s)

    def check_linear(b, x, w, y, residual=None, gated=False, out_type=BF16):
        xo = operand(b, x)
        z, off = product(xo, weights[w], None, op, out_type)
        if gated:
            z2, off2 = product(xo, weights["up"], None, op, out_type)
            v, off = act(z, "silu"), act_off(z, off, "silu")
            off, z = off * (np.abs(z2) + off2) + np.abs(v) * off2 + np.abs(v * z2) * 2.0**-24, v * z2
        if residual:
            z = z + d(b[residual])
            off = off + np.abs(z) * 2.0**-24
        assert np.all(np.abs(d(b[y]) - z) <= rounded(z, off, out_type)), (x, w, y)

    def check(b):
        scale = lambda n: b[n + "s"] if coded else None  # noqa: E731
        check_norm(b["x"], None, gamma[0], True, 1e-5, type_, op, b["n1"], None, scale("n1"))
        check_linear(b, "n1", "qkv", "qkv")
        check_norm(b["att"], None, None, False, 0, type_, op, b["a8"], None, scale("a8"))
        check_linear(b, "a8", "out", "mid", residual="x")
        check_norm(b["mid"], b["x"], gamma[1], True, 1e-5, type_, op, b["n2"], b["sum"], scale("n2"))
        check_linear(b, "n2", "gate", "h", gated=True)
        check_norm(b["h"], None, None, False, 0, type_, op, b["h8"], None, scale("h8"))
        check_linear(b, "h8", "down", "end", residual="sum")
        check_norm(b["tail"], None, gamma[2], True, 1e-5, type_, op, b["n3"], None, scale("n3"))
        check_linear(b, "n3", "head", "logits", out_type=F32)

    rng = np.random.default_rng(0)
    tokens = [list(rng.integers(0, vocab, n)) for n in prompt]
    one, graph = buffers([1, 1, 1]), None
    for i in range(steps + 1):
        rows = prompt if i == 0 else [1, 1, 1]
        b = buffers(rows) if i == 0 else one
        lens = [n + i for n in prompt]
        b["tok"].copy_(torch.tensor(sum(([*t[-r:]] for t, r in zip(tokens, rows)), [])))
        b["pos"].copy_(torch.tensor(np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)]), dtype=torch.int32))
        b["kv"].copy_(torch.tensor(lens, dtype=torch.int32))
        b["last"].copy_(torch.tensor(np.cumsum(rows) - 1))
        u = rng.random(3).astype(np.float32)
        b["u"].copy_(torch.from_numpy(u))
        torch.cuda.synchronize()
        if i == 0:
            step(b, rows)
        elif graph is None:
            with torch.cuda.stream(stream):
                step(b, rows)  # (what torch sets up at first use)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(b, rows)
            graph.replay()
        else:
            graph.replay()
        torch.cuda.synchronize()
        backend.check_device()
        check(b)
        logits = d(b["logits"])
        for s in range(3):
            want_id, _, gap = sample(logits[s], 1.0, 0, 1.0, 0.0, float(u[s]))
            assert gap <= 1e-11 or int(b["ids"][s]) == want_id
            tokens[s].append(int(b["ids"][s]))
