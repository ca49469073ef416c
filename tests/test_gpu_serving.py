"""Serving calls on the GPU against their definitions in 64 bits: rotary positions, the paged cache written and read, attention over it,
sampling, and a run of them together."""
import math

import numpy as np
import pytest
import torch

from mimir_framework_b200 import abi
from serving_ref import TOP, TORCH, Pages, attention, attention_bounds, half_step, sample

pytestmark = pytest.mark.gpu
F32, F16, BF16, I8, E4M3 = abi.T_F32, abi.T_F16, abi.T_BF16, abi.T_I8, abi.T_E4M3


def normal(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# ---- rotary positions ------------------------------------------------------------------------------------------------------------
def turned(x, pos, freq, rot, inter, m=1.0):
    angle = pos.astype(np.float64)[:, None] * freq
    c, s = m * np.cos(angle)[:, None], m * np.sin(angle)[:, None]
    y = x.copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("rows,heads,dim,rot,inter", [(1, 1, 2, 2, True), (3, 5, 64, 64, False), (17, 3, 128, 32, True), (5, 2, 80, 40, False), (700, 4, 256, 256, False),
                                                      (9, 3, 30, 6, False), (2, 7, 96, 96, True), (1300, 2, 24, 24, True), (40, 3, 48, 16, False)])
def test_rope(backend, rows, heads, dim, rot, inter, type_):
    x = normal(rows, heads, dim, seed=rows, dtype=TORCH[type_])
    pos = np.random.default_rng(rows).integers(-5, 3_000_000, rows).astype(np.int32)
    pos[0] = 0
    p = torch.from_numpy(pos).cuda()
    y = torch.full_like(x, float("nan"))
    strides = (heads * dim, dim)
    plan = backend.rope_plan(rot, interleaved=inter, magnitude=1.25)
    backend.dev_rope(plan, p.data_ptr(), x.data_ptr(), y.data_ptr(), rows, heads, dim, strides, strides, type_)
    freq = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
    xd = x.double().cpu().numpy()
    want = turned(xd, pos, freq, rot, inter, 1.25)
    # cosine and sine: their argument's and their own rounding and the magnitude's, 4 units of 2^-24 of 1.25; two products and a sum
    size = np.abs(turned(np.abs(xd), 0 * pos, freq, rot, inter)).max(-1, keepdims=True) * 2 * 1.25
    err = np.abs(y.double().cpu().numpy() - want)
    assert np.all(err <= size * 8 * 2.0**-24 + np.abs(want) * half_step(type_) * 1.001 + (2.0**-24 if type_ == F16 else 0))
    assert torch.equal(y[..., rot:], x[..., rot:])
    # in place, and back again
    z = x.clone()
    backend.dev_rope(plan, p.data_ptr(), z.data_ptr(), z.data_ptr(), rows, heads, dim, strides, strides, type_)
    assert torch.equal(z, y)
    back = backend.rope_plan(rot, interleaved=inter, magnitude=0.8, inverse=True)
    backend.dev_rope(back, p.data_ptr(), z.data_ptr(), z.data_ptr(), rows, heads, dim, strides, strides, type_)
    again = np.abs(z.double().cpu().numpy() - xd)
    assert np.all(again <= size * (16 * 2.0**-24 + 4 * half_step(type_)))


def test_rope_strides_and_neighbours(backend):
    """Queries and keys inside a wider projection, from an odd start, into another layout; nothing else is touched."""
    rows, heads, dim = 33, 6, 64
    wide = normal(rows, 3 * heads * dim + 5, seed=3)
    out = torch.full((heads, rows, dim + 3), -7.0, device="cuda")
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    plan = backend.rope_plan(32)
    src = wide[:, 3 : 3 + heads * dim]
    backend.dev_rope(plan, pos.data_ptr(), src.data_ptr(), out.data_ptr(), rows, heads, dim, (wide.stride(0), dim), (dim + 3, rows * (dim + 3)), F32)
    x = src.reshape(rows, heads, dim).double().cpu().numpy()
    want = turned(x, np.arange(rows), 10000.0 ** (-2.0 * np.arange(16) / 32), 32, False)
    assert np.abs(out[..., :dim].permute(1, 0, 2).double().cpu().numpy() - want).max() <= np.abs(x).max() * 2 * 10 * 2.0**-24
    assert (out[..., dim:] == -7.0).all()


# ---- cache ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("order", ["slot", "head"])
@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("cache", [F32, F16, BF16, I8, E4M3])
def test_cache_write_and_read(backend, cache, type_, order):
    for rows, kv, heads, dim, page in [([1], [1], 1, 8, 8), ([3, 0, 40, 1], [9, 5, 40, 130], 3, 80, 24), ([7, 5], [3, 64], 2, 256, 16)]:
        p = Pages(rows, kv, heads, dim, page, cache, order, seed=dim, gap=8)
        q = Pages(rows, kv, heads, dim, page, cache, order, seed=dim, gap=8)
        k, v = (normal(p.n_rows + 2, heads, dim + 8, seed=s, dtype=TORCH[type_])[..., :dim] for s in (1, 2))
        k[0, 0, :] = 0.0
        args = (type_, heads * (dim + 8), dim + 8)
        backend.dev_cache_write(p.cache(), p.batch(n_rows=p.n_rows + 2), k.data_ptr(), v.data_ptr(), *args)
        for s in range(len(kv)):
            n = min(rows[s], kv[s])  # (of more rows than keys the first have no place)
            if not n:
                continue
            for which, x in ((0, k), (1, v)):
                x = x[q.starts[s + 1] - n : q.starts[s + 1]]
                q.put(which, s, np.arange(kv[s] - n, kv[s]), torch.where(x == 0, torch.zeros_like(x), x))
        for a, b in zip(p.pool, q.pool):
            if cache in TOP:  # (the reference divides zeros by a zero scale)
                a, b = a.float().nan_to_num(0.0), b.float().nan_to_num(0.0)
                same = a == b
            else:
                same = (a == b) | (a.isnan() & b.isnan())
            assert same.all()
        if cache in TOP:
            for a, b in zip(p.scale, q.scale):
                assert ((a == b) | (a.isnan() & b.isnan())).all()
        # back out: what lies in the pages, code by code
        p.fill(seed=5)
        starts = np.concatenate([[0], np.cumsum([n + 2 for n in kv])]).astype(np.int32)
        o = torch.from_numpy(starts).cuda()
        got = [torch.full((int(starts[-1]) + 1, heads, dim + 8), -7.0, dtype=TORCH[type_], device="cuda") for _ in range(2)]
        backend.dev_cache_read(p.cache(), p.batch(), o.data_ptr(), int(starts[-1]) + 1, got[0].data_ptr(), got[1].data_ptr(), *args)
        backend.check_device()
        for which in range(2):
            for s, n in enumerate(kv):
                x = torch.from_numpy(p.get(which, s)).float().to(TORCH[type_])  # (one fp32 product, one rounding)
                rows_of = got[which][starts[s] : starts[s + 1]]
                assert torch.equal(rows_of[:n, :, :dim].cpu(), x)
                assert (rows_of[n:] == -7.0).all() and (rows_of[..., dim:] == -7.0).all()
            assert (got[which][-1] == -7.0).all()


@pytest.mark.parametrize("cache,type_", [(F16, F16), (E4M3, BF16)])
def test_cache_of_many_heads_and_sequences(backend, cache, type_):
    """More heads than a block moves at once, more sequences than it keeps the starts of."""
    rng = np.random.default_rng(1)
    for n_seqs, heads, dim in ((3, 70, 64), (1100, 2, 16)):
        rows = [int(v) for v in rng.integers(0, 3, n_seqs)]
        kv = [n + int(v) for n, v in zip(rows, rng.integers(0, 9, n_seqs))]
        p, q = (Pages(rows, kv, heads, dim, 8, cache, seed=2) for _ in range(2))
        k, v = (normal(p.n_rows, heads, dim, seed=s, dtype=TORCH[type_]) for s in (1, 2))
        backend.dev_cache_write(p.cache(), p.batch(), k.data_ptr(), v.data_ptr(), type_, heads * dim, dim)
        for s in range(n_seqs):
            if rows[s]:
                for which, x in ((0, k), (1, v)):
                    q.put(which, s, np.arange(kv[s] - rows[s], kv[s]), x[q.starts[s] : q.starts[s + 1]])
        for a, b in zip(p.pool + p.scale, q.pool + q.scale):
            if a is not None:
                a, b = a.float(), b.float()
                assert ((a == b) | (a.isnan() & b.isnan())).all()
        p.fill(seed=4)
        starts = np.concatenate([[0], np.cumsum(kv)]).astype(np.int32)
        o = torch.from_numpy(starts).cuda()
        got = [torch.full((int(starts[-1]), heads, dim), -7.0, dtype=TORCH[type_], device="cuda") for _ in range(2)]
        backend.dev_cache_read(p.cache(), p.batch(), o.data_ptr(), int(starts[-1]), got[0].data_ptr(), got[1].data_ptr(), type_, heads * dim, dim)
        backend.check_device()
        for which in range(2):
            want = np.concatenate([p.get(which, s) for s in range(n_seqs)])
            assert torch.equal(got[which].cpu(), torch.from_numpy(want).float().to(TORCH[type_]))


@pytest.mark.parametrize("cache", [I8, E4M3])
def test_codes_of_values_that_are_not_finite(backend, cache):
    p = Pages([4], [4], 1, 8, 8, cache)
    x = torch.tensor([[1.0, -2.0, float("inf"), -float("inf"), 0.5, 0, 0, 0], [float("nan"), 4.0, 1, 1, 1, 1, 1, 1], [float("inf")] * 8, [1e-44] * 8],
                     device="cuda").view(4, 1, 8)
    backend.dev_cache_write(p.cache(), p.batch(), x.data_ptr(), x.data_ptr(), F32, 8, 8)
    backend.check_device()
    page = int(p.table[0, 0])
    codes, scales = p.pool[0][page, :4, 0].float().cpu(), p.scale[0][page, 0, :4].cpu()
    top = TOP[cache]
    assert scales[0] == torch.tensor(2.0) * torch.tensor(1 / top) and codes[0, 1] == -top and codes[0, 2] == top and codes[0, 3] == -top
    assert codes[1, 1] == top and (codes[1, 0] == 0 if cache == I8 else codes[1, 0].isnan())
    assert scales[2] == 0 and (codes[2] == 0).all()
    assert scales[3] == 0 and (codes[3] == 0).all()  # 1e-44 / 127 is no fp32 number but zero


# ---- attention --------------------------------------------------------------------------------------------------------------------
PAIRS = [(F32, F32), (F16, F32), (F16, F16), (F16, BF16), (BF16, BF16), (I8, F32), (I8, F16), (I8, BF16), (E4M3, F32), (E4M3, F16), (E4M3, BF16)]


def attend(backend, p, heads, type_, causal=True, window=0, seed=7, spread=1.0, stream=0, gap=0, change=None, extra_rows=0, **batch):
    q = normal(p.n_rows + extra_rows, heads, p.dim + gap, seed=seed, scale=spread, dtype=TORCH[type_])
    out = torch.full_like(q, -7.0)
    lse = torch.full((p.n_rows + extra_rows, heads), -7.0, device="cuda")
    cache, b = p.cache(**(change or {})), p.batch(n_rows=p.n_rows + extra_rows, **batch)
    a = backend.paged_attention(q.data_ptr(), out.data_ptr(), type_, heads, heads * (p.dim + gap), p.dim + gap, heads * (p.dim + gap), p.dim + gap,
                                1 / math.sqrt(p.dim), causal, window, lse.data_ptr())
    size = backend.paged_attention_workspace(cache, b, a)
    ws = torch.full((size + 16,), 255, dtype=torch.uint8, device="cuda")
    if size:
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
    torch.cuda.synchronize()
    backend.dev_paged_attention(cache, b, a, stream)
    torch.cuda.synchronize()
    assert (ws[size:] == 255).all()
    return q, out, lse


def check_attention(p, q, out, lse, type_, causal, window):
    n = p.n_rows
    want, want_lse, weight, reach = attention(p, q[:n, :, : p.dim].double().cpu().numpy(), 1 / math.sqrt(p.dim), causal, window)
    # bf16 and e4m3 / i8 tensors meet bf16 or half terms; the bound goes by the result's type
    chunk = type_ != F32 and q.shape[1] // p.heads * max(p.rows, default=0) > 32
    bound, lse_bound = attention_bounds(want, weight, reach, p.dim, max(p.kv, default=0), BF16 if p.type == BF16 else type_, chunk,
                                         type_ == BF16 and p.type != BF16)
    err = np.abs(out[:n, :, : p.dim].double().cpu().numpy() - want)
    assert np.all(err <= bound), f"{np.max(err / np.maximum(bound, 1e-300))} of the bound"
    got = lse[:n].double().cpu().numpy()
    empty = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(got), empty)
    got, want_lse, lse_bound = got[~empty], want_lse[~empty], lse_bound[~empty]
    assert np.all(np.abs(got - want_lse) <= lse_bound + np.abs(want_lse) * 2.0**-22)
    assert (out[:n, :, : p.dim].float().cpu().numpy()[empty] == 0).all()
    assert (out[n:] == -7.0).all() and (out[..., p.dim :] == -7.0).all() and (lse[n:] == -7.0).all()


@pytest.mark.parametrize("cache,type_", PAIRS)
@pytest.mark.parametrize("rows,kv,kv_heads,group,dim,page,causal,window", [
    ([1], [1], 1, 1, 8, 8, True, 0),                                     # one key
    ([1, 1, 1], [33, 257, 1], 2, 4, 64, 24, True, 0),                    # pages that end inside a block of keys
    ([2, 0, 5, 1], [40, 7, 3, 130], 3, 5, 80, 16, True, 0),              # no rows; more rows than keys: rows that see nothing
    ([1, 0, 1], [0, 0, 20], 1, 8, 128, 8, False, 0),                     # no keys at all
    ([37, 20], [100, 20], 1, 3, 32, 32, True, 0),                        # chunks of a prompt, a whole one
    ([33, 3], [150, 64], 2, 2, 128, 16, True, 17),                       # a window narrower than the chunk
    ([5, 1], [90, 300], 1, 16, 256, 64, False, 40),                      # a window, not causal
    ([130], [200], 2, 1, 192, 40, True, 0)])
def test_attention(backend, rows, kv, kv_heads, group, dim, page, causal, window, cache, type_):
    order = "head" if dim % 3 else "slot"
    p = Pages(rows, kv, kv_heads, dim, page, cache, order, seed=dim, gap=16 if dim == 64 else 0)
    p.fill()
    heads = kv_heads * group
    q, out, lse = attend(backend, p, heads, type_, causal, window, gap=8 if dim == 80 else 0, extra_rows=2)
    backend.check_device()
    check_attention(p, q, out, lse, type_, causal, window)


@pytest.mark.parametrize("cache,type_", PAIRS)
@pytest.mark.parametrize("rows,kv,kv_heads,group,dim,page,causal,window", [
    ([65], [65], 1, 1, 64, 16, True, 0),                                   # a tile mostly empty
    ([33], [33], 1, 1, 64, 16, True, 0),                                   # one row over the rows of few
    ([257, 1, 64, 130], [300, 700, 64, 130], 1, 1, 128, 24, True, 0),      # many and few rows in one batch
    ([257, 1, 32, 33, 130], [300, 700, 64, 50, 130], 1, 1, 128, 24, True, 0),
    ([200, 90], [900, 50], 2, 2, 64, 8, True, 0),                          # more rows than keys
    ([100, 0, 70], [0, 40, 71], 1, 4, 96, 128, False, 0),                  # no keys; no rows; not causal
    ([300], [1111], 1, 1, 128, 64, True, 77),                              # a window narrower than a tile
    ([129], [2000], 1, 2, 256, 16, True, 300),
    ([80], [9000], 1, 2, 256, 64, True, 0),                                # few tiles, many keys: parts in the workspace
    ([80, 5], [9000, 3000], 1, 2, 40, 56, False, 0)])
def test_attention_of_chunks(backend, rows, kv, kv_heads, group, dim, page, causal, window, cache, type_):
    p = Pages(rows, kv, kv_heads, dim, page, cache, "head" if group == 2 else "slot", seed=dim, gap=24 if dim == 96 else 0)
    p.fill()
    q, out, lse = attend(backend, p, kv_heads * group, type_, causal, window, gap=8 if dim == 40 else 0, extra_rows=3)
    backend.check_device()
    check_attention(p, q, out, lse, type_, causal, window)


@pytest.mark.parametrize("cache,type_,dim", [(BF16, BF16, 256), (I8, F16, 256), (E4M3, F32, 64), (F16, F32, 128)])
def test_chunks_whose_score_tiles_alternate_many_times_over(backend, cache, type_, dim):
    """Many blocks' ends: none may wait for a product that is through already."""
    p = Pages([512] * 8, [2048] * 8, 4, dim, 64, cache, seed=5)
    p.fill()
    outs = []
    q, out, lse = attend(backend, p, 8, type_)
    outs.append(out.clone())
    a = backend.paged_attention(q.data_ptr(), out.data_ptr(), type_, 8, 8 * dim, dim, 8 * dim, dim, 1 / math.sqrt(dim), lse=lse.data_ptr())
    for _ in range(100):
        backend.dev_paged_attention(p.cache(), p.batch(), a)
    backend.check_device()
    assert torch.equal(outs[0], out)


@pytest.mark.parametrize("cache,type_", [(BF16, BF16), (F16, F32), (I8, F16)])
def test_attention_of_many_sequences(backend, cache, type_):
    """More sequences than a warp has lanes, of no, few and many rows in no order; rows behind the last one stay."""
    rng = np.random.default_rng(4)
    rows = [int(rng.choice([0, 1, 1, 1, 16, 17, 40, 150])) for _ in range(83)] + [0, 0, 133]
    kv = [int(max(0, r + rng.integers(-3, 90))) for r in rows]
    p = Pages(rows, kv, 2, 64, 16, cache, seed=8)
    p.fill()
    q, out, lse = attend(backend, p, 4, type_, window=50, extra_rows=5)
    backend.check_device()
    check_attention(p, q, out, lse, type_, True, 50)


@pytest.mark.parametrize("cache,type_", [(BF16, BF16), (F16, F32), (I8, F16), (F32, F32)])
@pytest.mark.parametrize("rows,group", [([1, 1, 0, 1], 48), ([1], 71), ([2, 1], 40)])
def test_attention_of_one_key_head_for_many(backend, rows, group, cache, type_):
    """A single token's heads alone are more rows than a tile of few."""
    p = Pages(rows, [900, 33, 5, 1][: len(rows)], 1, 64, 16, cache, seed=8)
    p.fill()
    q, out, lse = attend(backend, p, group, type_)
    backend.check_device()
    check_attention(p, q, out, lse, type_, True, 0)


def test_attention_with_the_largest_window_and_limits(backend):
    """Numbers at the end of their range: a window that nothing fills is none, limits are limits."""
    most = 2**31 - 1
    for rows in ([3, 1], [60, 2]):
        p = Pages(rows, [50, 40], 1, 64, 16, F16, seed=8)
        p.fill()
        q, out, lse = attend(backend, p, 2, F16, window=most)
        check_attention(p, q, out, lse, F16, True, 0)
        got = out.clone()
        q, out, lse = attend(backend, p, 2, F16, window=most, max_kv=most, max_rows=most)
        backend.check_device()
        check_attention(p, q, out, lse, F16, True, 0)


@pytest.mark.parametrize("rows", [[1, 2], [140, 3]])
@pytest.mark.parametrize("cache,type_", [(BF16, BF16), (F16, F16), (E4M3, BF16), (I8, F32)])
def test_attention_over_large_pages(backend, rows, cache, type_):
    for page, order in ((256, "head"), (1000, "slot")):
        p = Pages(rows, [1300, 999], 1, 128, page, cache, order, seed=3)
        p.fill()
        q, out, lse = attend(backend, p, 2, type_)
        backend.check_device()
        check_attention(p, q, out, lse, type_, True, 0)


@pytest.mark.parametrize("rows,kv", [([2, 1], [15000, 2]), ([90, 1, 3], [6000, 4000, 70]), ([300, 40], [310, 7000])])
def test_attention_on_two_streams_and_captured(backend, rows, kv):
    """Two batches at once, each with its workspace, and a captured call that is replayed over other lengths and pages."""
    ps = [Pages(rows, kv, 1, 64, 16, F16, seed=s) for s in (1, 2)]
    calls, keep = [], []
    for i, p in enumerate(ps):
        p.fill(seed=i)
        q = normal(p.n_rows, 2, 64, seed=i, dtype=torch.float16)
        out, lse = torch.full_like(q, -7.0), torch.full((p.n_rows, 2), -7.0, device="cuda")
        a = backend.paged_attention(q.data_ptr(), out.data_ptr(), F16, 2, 128, 64, 128, 64, 0.125, lse=lse.data_ptr())
        ws = torch.full((backend.paged_attention_workspace(p.cache(), p.batch(), a) + 16,), 255, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        calls.append(a)
        keep.append((q, out, lse, ws))
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(5):
        for p, a, s in zip(ps, calls, streams):
            backend.dev_paged_attention(p.cache(), p.batch(), a, s.cuda_stream)
    torch.cuda.synchronize()
    backend.check_device()
    for p, (q, out, lse, _) in zip(ps, keep):
        check_attention(p, q, out, lse, F16, True, 0)
    p, a, (q, out, lse, _) = ps[0], calls[0], keep[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        backend.dev_paged_attention(p.cache(), p.batch(), a, streams[0].cuda_stream)
    # fewer rows in each sequence, in other places: the rest of the rows stay
    r = Pages([(n + 1) // 2 for n in rows], [n - 1 for n in kv], 1, 64, 16, F16, seed=5, spare=0)
    r.table = np.where(r.table >= 0, r.table + 1, r.table)[:, : p.width]
    r.n_pages, r.pool, r.width = p.n_pages, p.pool, p.width
    r.table = np.pad(r.table, ((0, 0), (0, p.width - r.table.shape[1])), constant_values=-77)
    r.fill(seed=9)
    for here, new in zip(p.dev, (r.starts, r.kv, r.table)):
        here.copy_(torch.from_numpy(np.asarray(new, np.int32)))
    out.fill_(-7.0)
    lse.fill_(-7.0)
    graph.replay()
    torch.cuda.synchronize()
    backend.check_device()
    check_attention(r, q, out, lse, F16, True, 0)


@pytest.mark.parametrize("cache,type_", [(BF16, BF16), (E4M3, F16), (F16, BF16)])
def test_chunks_with_a_negative_scale_a_bad_page_and_large_scores(backend, cache, type_):
    p = Pages([150, 70], [400, 90], 2, 64, 16, cache, seed=2)
    p.fill(spread=2.0)
    q, out, lse = attend(backend, p, 4, type_, spread=20.0)
    check_attention(p, q, out, lse, type_, True, 0)
    a = backend.paged_attention(q.data_ptr(), out.data_ptr(), type_, 4, 256, 64, 256, 64, -0.02, lse=lse.data_ptr())
    backend.dev_paged_attention(p.cache(), p.batch(), a)
    want, want_lse, weight, reach = attention(p, q.double().cpu().numpy(), -0.02, True, 0)
    bound, lse_bound = attention_bounds(want, weight, reach, 64, 400, BF16 if cache == BF16 else type_, True)
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound)
    # keys 32 .. 47 of the first sequence are in no page
    bad = p.dev[2].clone()
    bad[0, 2] = -1
    backend.dev_paged_attention(p.cache(), p.batch(page_table=bad.data_ptr()), a)
    with pytest.raises(backend.MimirB200Error, match="page number"):
        backend.check_device()
    kept = [j for j in range(400) if not 32 <= j < 48]
    r = Pages([150, 70], [384, 90], 2, 64, 16, cache, seed=3)
    for w in range(2):
        r.put(w, 0, np.arange(384), torch.from_numpy(p.get(w, 0)[kept]).cuda())
        r.put(w, 1, np.arange(90), torch.from_numpy(p.get(w, 1)).cuda())
    for w in range(2):  # (stored as the same codes and scales: nothing is rounded again)
        assert np.abs(r.get(w, 0) - p.get(w, 0)[kept]).max() <= 2.0**-20 * np.abs(p.get(w, 0)).max()
    want, _, weight, reach = attention(r, q.double().cpu().numpy(), -0.02, True, 0)
    bound, _ = attention_bounds(want, weight, reach, 64, 400, BF16 if cache == BF16 else type_, True)
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound + 2.0**-18 * np.abs(weight))


@pytest.mark.parametrize("cache,type_", [(BF16, BF16), (F16, F32), (E4M3, BF16), (I8, F16)])
def test_attention_of_long_sequences(backend, cache, type_):
    """Few tiles and many keys: parts in the workspace; and in a cache whose offsets pass 32 bits."""
    p = Pages([1, 2], [20000, 9001], 1, 64, 64, cache, seed=4)
    p.fill(spread=2.0)
    q, out, lse = attend(backend, p, 4, type_)
    backend.check_device()
    check_attention(p, q, out, lse, type_, True, 0)


def test_attention_of_far_pages(backend):
    p = Pages([1], [300], 2, 128, 16, I8, seed=1, spare=3)
    p.fill()
    # 17 of its pages 2^28 elements apart; only those that are used are ever touched
    stride, pages = 1 << 28, 17
    big = [torch.empty(pages * stride + 4096, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.full((pages + 1, 2, 16), float("nan"), device="cuda") for _ in range(2)]
    table = torch.full_like(p.dev[2], -77)
    for j in range(pages):
        to = pages if j == 7 else j
        table[0, j] = to
        for w in range(2):
            big[w][to * stride : to * stride + 4096] = p.pool[w][int(p.table[0, j])].reshape(-1)
            scales[w][to] = p.scale[w][int(p.table[0, j])]
    p.kv = [pages * 16 - 3]
    p.dev[1].fill_(p.kv[0])
    p.dev[2] = table
    change = dict(k=big[0].data_ptr(), v=big[1].data_ptr(), k_scale=scales[0].data_ptr(), v_scale=scales[1].data_ptr(), n_pages=pages + 1, page_stride=stride)
    q, out, lse = attend(backend, p, 4, F32, change=change)
    backend.check_device()
    check_attention(p, q, out, lse, F32, True, 0)


@pytest.mark.parametrize("cache,type_", [(F16, F16), (BF16, BF16), (F16, F32), (F32, F32), (E4M3, F32)])
def test_attention_of_large_and_small_values(backend, cache, type_):
    """Scores in the hundreds, where one key has nearly everything; queries far from one."""
    p = Pages([3, 1], [70, 200], 2, 64, 16, cache, seed=2)
    p.fill(spread=3.0)
    q, out, lse = attend(backend, p, 4, type_, spread=30.0)
    check_attention(p, q, out, lse, type_, True, 0)
    q, out, lse = attend(backend, p, 4, type_, spread=1e-3)
    check_attention(p, q, out, lse, type_, True, 0)


def test_scales_of_any_size(backend):
    """Codes whose scales span many powers of two from key to key."""
    for cache in (I8, E4M3):
        p = Pages([2], [90], 1, 64, 16, cache, seed=6)
        g = torch.Generator(device="cuda")
        g.manual_seed(3)
        x = torch.randn(90, 1, 64, generator=g, device="cuda")
        p.put(0, 0, np.arange(90), x)
        p.put(1, 0, np.arange(90), x * torch.exp2(torch.arange(90, device="cuda") % 41 - 20.0)[:, None, None])
        q, out, lse = attend(backend, p, 2, F32)
        want, _, weight, reach = attention(p, q.double().cpu().numpy(), 1 / 8, True, 0)
        # a probability times its scale is two halves of one block's largest scale: below 2^-24 of that it is zero
        bound, _ = attention_bounds(want, weight, reach, 64, 90, F32)
        top = np.abs(p.get(1, 0)).max()
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound + 90 * 2.0**-23 * top)


def test_bad_numbers_are_reported_and_left_out(backend):
    p = Pages([1, 1, 1, 1], [40, 40, 40, 40], 2, 64, 16, F16, seed=9)
    p.fill()
    # sequence 1: a page outside the cache; 2: more keys than max_kv; 3: rows that run past the tensors
    p.dev[2][1, 1] = p.n_pages
    p.dev[1][2] = 41
    p.dev[0][4] = 5
    q, out, lse = attend(backend, p, 4, F16)
    with pytest.raises(backend.MimirB200Error) as e:
        backend.check_device()
    assert e.value.status == abi.E_INVALID and "page number" in str(e.value) and "key count" in str(e.value) and "row ranges" in str(e.value)
    backend.check_device()  # (cleared)
    want, want_lse, weight, reach = attention(p, q.double().cpu().numpy(), 1 / 8, True, 0)
    bound, _ = attention_bounds(want, weight, reach, 64, 40, F16)
    assert np.all(np.abs(out[0].double().cpu().numpy() - want[0]) <= bound[0])
    assert (out[2] == 0).all() and torch.isneginf(lse[2]).all() and (out[3] == -7.0).all()
    # the same by the cache's calls: only what fits is written
    k = normal(4, 2, 64, dtype=torch.float16)
    before = [t.clone() for t in p.pool]
    p.dev[1].fill_(17)
    p.dev[1][2] = 41
    backend.dev_cache_write(p.cache(), p.batch(), k.data_ptr(), k.data_ptr(), F16, 128, 64)
    with pytest.raises(backend.MimirB200Error):
        backend.check_device()
    for old, new in zip(before, p.pool):
        changed = (old.view(torch.int16) != new.view(torch.int16)).flatten(1).any(1).nonzero().flatten().tolist()
        assert changed == [int(p.table[0, 1])]
    starts = torch.tensor([0, 40, 80, 120, 161], dtype=torch.int32, device="cuda")
    o = torch.full((160, 2, 64), -7.0, dtype=torch.float16, device="cuda")
    p.dev[1].fill_(40)
    backend.dev_cache_read(p.cache(), p.batch(), starts.data_ptr(), 160, o.data_ptr(), o.data_ptr(), F16, 128, 64)
    with pytest.raises(backend.MimirB200Error):
        backend.check_device()
    assert (o[56:72] == -7.0).all() and (o[120:] == -7.0).all() and (o[:56] != -7.0).any(1).all()


def test_refusals_of_pointers(backend):
    p = Pages([1], [40], 2, 64, 16, I8, seed=9)
    x = normal(1, 4, 64, dtype=torch.float16)
    host = torch.zeros(4096, dtype=torch.float16)
    att = backend.paged_attention(x.data_ptr(), x.data_ptr(), F16, 4, 256, 64, 256, 64, 0.125)
    plan = backend.rope_plan(64)
    u = torch.zeros(1, device="cuda")
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    for f in (lambda: backend.dev_paged_attention(p.cache(k=host.data_ptr()), p.batch(), att), lambda: backend.dev_paged_attention(p.cache(v_scale=None), p.batch(), att),
              lambda: backend.dev_paged_attention(p.cache(), p.batch(kv_len=None), att),
              lambda: backend.dev_paged_attention(p.cache(k=p.pool[0].data_ptr() + 8), p.batch(), att),
              lambda: backend.dev_paged_attention(p.cache(), p.batch(), backend.paged_attention(x.data_ptr() + 2, x.data_ptr(), F16, 4, 256, 64, 256, 64, 0.125)),
              lambda: backend.dev_cache_write(p.cache(), p.batch(), host.data_ptr(), x.data_ptr(), F16, 128, 64),
              lambda: backend.dev_cache_read(p.cache(), p.batch(), 0, 1, x.data_ptr(), x.data_ptr(), F16, 128, 64),
              lambda: backend.dev_rope(plan, p.dev[1].data_ptr(), x.data_ptr(), host.data_ptr(), 1, 4, 64, (256, 64), (256, 64), F16),
              lambda: backend.dev_rope(plan, p.dev[1].data_ptr(), x.data_ptr() + 1, x.data_ptr(), 1, 1, 64, (256, 64), (256, 64), F16),
              lambda: backend.dev_sample_rows(x.data_ptr(), F16, 1, 256, 256, None, None, None, None, None, ids.data_ptr()),
              lambda: backend.dev_sample_rows(x.data_ptr(), F16, 1, 256, 256, host.data_ptr(), None, None, None, u.data_ptr(), ids.data_ptr())):
        with pytest.raises(backend.MimirB200Error) as e:
            f()
        assert e.value.status in (abi.E_INVALID, abi.E_UNSUPPORTED)
    # few long sequences need a workspace
    q = Pages([1], [40000], 1, 64, 64, F16)
    a = backend.paged_attention(x.data_ptr(), x.data_ptr(), F16, 4, 256, 64, 256, 64, 0.125)
    assert backend.paged_attention_workspace(q.cache(), q.batch(), a) > 0
    with pytest.raises(backend.MimirB200Error, match="workspace"):
        backend.dev_paged_attention(q.cache(), q.batch(), a)
    # empty batches are no work
    backend.dev_paged_attention(p.cache(), p.batch(n_seqs=0), att)
    backend.dev_paged_attention(p.cache(), p.batch(n_rows=0), att)
    backend.dev_cache_write(p.cache(), p.batch(n_rows=0), None, None, F16, 128, 64)
    backend.check_device()


def test_refusals_of_words_off_their_boundary(backend):
    p = Pages([1], [40], 2, 64, 16, I8, seed=9)
    x = normal(1, 4, 64, dtype=torch.float16)
    room = torch.zeros(64, dtype=torch.int32, device="cuda")
    odd, ok = room.data_ptr() + 2, room.data_ptr()
    att = backend.paged_attention(x.data_ptr(), x.data_ptr(), F16, 4, 256, 64, 256, 64, 0.125)
    lse = backend.paged_attention(x.data_ptr(), x.data_ptr(), F16, 4, 256, 64, 256, 64, 0.125, lse=odd)
    for f in (lambda: backend.dev_paged_attention(p.cache(), p.batch(row_start=odd), att), lambda: backend.dev_paged_attention(p.cache(), p.batch(kv_len=odd), att),
              lambda: backend.dev_paged_attention(p.cache(), p.batch(page_table=odd), att), lambda: backend.dev_paged_attention(p.cache(), p.batch(), lse),
              lambda: backend.dev_cache_write(p.cache(), p.batch(kv_len=odd), x.data_ptr(), x.data_ptr(), F16, 128, 64),
              lambda: backend.dev_cache_read(p.cache(), p.batch(), odd, 1, x.data_ptr(), x.data_ptr(), F16, 128, 64),
              lambda: backend.dev_rope(backend.rope_plan(64), odd, x.data_ptr(), x.data_ptr(), 1, 4, 64, (256, 64), (256, 64), F16),
              lambda: backend.dev_sample_rows(x.data_ptr(), F16, 1, 256, 256, None, None, None, None, odd, ok),
              lambda: backend.dev_sample_rows(x.data_ptr(), F16, 1, 256, 256, None, odd, None, None, ok, ok),
              lambda: backend.dev_sample_rows(x.data_ptr(), F16, 1, 256, 256, None, None, None, None, ok, odd)):
        with pytest.raises(backend.MimirB200Error, match="aligned") as e:
            f()
        assert e.value.status == abi.E_INVALID
    backend.check_device()


# ---- sampling -------------------------------------------------------------------------------------------------------------------------
def draw(backend, x, t=None, k=None, p=None, m=None, u=None, type_=F32, stride=None):
    rows, n = x.shape
    ids, logp = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda"), torch.full((rows + 1,), -7.0, device="cuda")
    at = lambda v: None if v is None else v.data_ptr()  # noqa: E731
    backend.dev_sample_rows(x.data_ptr(), type_, rows, n, stride or x.stride(0), at(t), at(k), at(p), at(m), u.data_ptr(), ids.data_ptr(), logp.data_ptr())
    torch.cuda.synchronize()
    assert ids[-1] == -7 and logp[-1] == -7.0
    return ids[:-1].cpu().numpy(), logp[:-1].double().cpu().numpy()


def check_sample(x, t, k, p, m, u, ids, logp):
    xd = x.double().cpu().numpy()
    each = [v.double().cpu().numpy() if v is not None else np.full(len(xd), d) for v, d in ((t, 1.0), (k, 0), (p, 1.0), (m, 0.0), (u, 0.0))]
    for r in range(len(xd)):
        want, lp, gap = sample(xd[r], each[0][r], int(each[1][r]), each[2][r], each[3][r], each[4][r])
        # both sides' sums are exact to better than 1e-11: on a border nearer than that either neighbour is right
        if gap > 1e-11:
            assert ids[r] == want, (r, ids[r], want)
            if np.isfinite(lp):
                assert abs(logp[r] - lp) <= 2.0**-22 * max(1.0, abs(lp))
            else:
                assert logp[r] == lp


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (7, 31), (5, 1000), (2, 1025), (9, 32000), (2, 50257), (3, 151936), (300, 700)])
def test_sampling(backend, rows, n, type_):
    x = normal(rows, n + 3, seed=n, scale=3.0, dtype=TORCH[type_])[:, 1 : n + 1]  # (rows apart, an odd start)
    g = np.random.default_rng(n)
    for k, p, m in [(0, 1.0, 0.0), (1, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (50, 0.7, 0.01), (n, 0.0, 0.0), (0, 0.999, 2.0), (-3, 1.5, -1.0)]:
        u = torch.from_numpy(g.random(rows).astype(np.float32)).cuda()
        t = torch.from_numpy(g.uniform(0.3, 2.0, rows).astype(np.float32)).cuda()
        kk, pp, mm = torch.full((rows,), k, dtype=torch.int32, device="cuda"), torch.full((rows,), p, device="cuda"), torch.full((rows,), m, device="cuda")
        ids, logp = draw(backend, x, t, kk, pp, mm, u, type_)
        check_sample(x, t, kk, pp, mm, u, ids, logp)
    ids, logp = draw(backend, x, None, None, None, None, u, type_)
    check_sample(x, None, None, None, None, u, ids, logp)


@pytest.mark.parametrize("n,type_", [(400_003, F32), (1_500_001, BF16)])
def test_sampling_of_rows_beyond_shared_memory(backend, n, type_):
    x = normal(2, n, seed=n, scale=3.0, dtype=TORCH[type_])
    g = np.random.default_rng(n)
    for k, p, m in [(0, 1.0, 0.0), (40, 0.9, 0.0), (5000, 0.8, 0.0), (0, 0.95, 0.02), (0, 0.5, 0.0), (n - 7, 0.999, 0.0)]:
        u = torch.from_numpy(g.random(2).astype(np.float32)).cuda()
        kk, pp, mm = torch.full((2,), k, dtype=torch.int32, device="cuda"), torch.full((2,), p, device="cuda"), torch.full((2,), m, device="cuda")
        ids, logp = draw(backend, x, None, kk, pp, mm, u, type_)
        check_sample(x, None, kk, pp, mm, u, ids, logp)


@pytest.mark.parametrize("rows,n,type_", [(200, 1000, F32), (96, 32000, BF16), (40, 151936, F16)])
def test_sampling_by_mass_and_by_least_share(backend, rows, n, type_):
    """min_p leaves a few or many, and top_p takes some of them or none; shares that meet the border exactly."""
    x = normal(rows, n, seed=n + 1, scale=2.5, dtype=TORCH[type_])
    x[::7] = x[::7].round() / 2  # (many equals)
    x[1] = 0.0
    x[2, 3:] = -20.0
    g = np.random.default_rng(n)
    for _ in range(4):
        u, t, p, m = (torch.from_numpy(v.astype(np.float32)).cuda() for v in (g.random(rows), g.uniform(0.3, 2.0, rows), 1 - 10 ** g.uniform(-3, -0.2, rows), 10 ** g.uniform(-4, -0.2, rows)))
        p[1], p[2], p[3] = 0.5, 0.25, 0.0
        ids, logp = draw(backend, x, t, None, p, m, u, type_)
        check_sample(x, t, None, p, m, u, ids, logp)


def test_sampling_with_parameters_that_are_no_numbers(backend):
    """Not a number: the largest logit (temperature), all (top_p, min_p), the first that stays (uniform)."""
    x = normal(6, 2000, seed=3, scale=2.0)
    u, ones = torch.full((6,), 0.4, device="cuda"), torch.ones(6, device="cuda")
    nan = torch.full((6,), float("nan"), device="cuda")
    ids, _ = draw(backend, x, nan, None, None, None, u)
    assert np.array_equal(ids, x.argmax(1).cpu().numpy())
    want = draw(backend, x, ones, None, None, None, u)
    for got in (draw(backend, x, ones, None, nan, None, u), draw(backend, x, ones, None, None, nan, u)):
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    ids, _ = draw(backend, x, ones, torch.full((6,), 3, dtype=torch.int32, device="cuda"), None, None, nan)
    assert np.array_equal(ids, x.topk(3, 1).indices.min(1).values.cpu().numpy())


def test_sampling_of_equal_and_absent_logits(backend):
    inf, nan = float("inf"), float("nan")
    n = 3000
    x = torch.zeros(12, n, device="cuda")
    x[1] = -inf
    x[2] = nan
    x[3, 100] = inf
    x[3, 7] = inf
    x[4, ::2] = -inf
    x[5] = torch.arange(n, device="cuda") % 3  # (many of the largest)
    x[6, 5:] = -inf
    x[7] = -1e38
    x[8, 1] = 3e38
    x[9, ::3] = nan
    x[10] = -0.0
    x[10, 1::2] = 0.0
    x[11] = torch.linspace(-1e-38, 1e-38, n, device="cuda")
    rows = len(x)
    for k, p, t in [(0, 1.0, 1.0), (10, 1.0, 1.0), (0, 0.5, 1.0), (999, 0.25, 0.7), (1, 1.0, 1.0), (5, 0.0, 1.0), (0, 1.0, 0.0), (0, 1.0, -1.0), (2500, 0.9, inf)]:
        for uu in (0.0, 0.37, 1.0 - 2.0**-24):
            u, tt = torch.full((rows,), uu, device="cuda"), torch.full((rows,), t, device="cuda")
            kk, pp = torch.full((rows,), k, dtype=torch.int32, device="cuda"), torch.full((rows,), p, device="cuda")
            ids, logp = draw(backend, x, tt, kk, pp, None, u)
            check_sample(x, tt, kk, pp, None, u, ids, logp)
    assert ids[1] == -1 and ids[2] == -1 and ids[3] == 7


def test_sampling_follows_the_shares(backend):
    """Every token comes up for as much of the random numbers as its share: the numbers in the middle of each share's stretch give it."""
    n = 500
    x = normal(1, n, seed=5, scale=2.0)
    w = np.exp(x.double().cpu().numpy()[0])
    edges = np.concatenate([[0.0], np.cumsum(w) / w.sum()])
    mid = ((edges[1:] + edges[:-1]) / 2).astype(np.float32)
    sure = (np.diff(edges) > 4 * 2.0**-24)
    u = torch.from_numpy(mid).cuda()
    ids, _ = draw(backend, x.expand(n, n).contiguous(), None, None, None, None, u)
    assert np.array_equal(ids[sure], np.arange(n)[sure]) and sure.sum() > n // 2


# ---- together -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", [F16, I8])
def test_generation_of_a_small_batch(backend, cache):
    """A prompt's chunk and then single tokens: rotary positions on queries and keys, the cache written, attention over it, logits and a token;
    the steps are captured once and replayed.  Every step's attention is held against the definition over what the cache then holds."""
    heads, kv_heads, dim, page, vocab = 6, 2, 64, 16, 300
    prompt, steps = [20, 5, 33], 4
    p = Pages(prompt, [n + steps for n in prompt], kv_heads, dim, page, cache, seed=3)
    wide = (heads + 2 * kv_heads) * dim
    table = normal(vocab, wide, seed=1)  # a token's projection
    head = normal(heads * dim, vocab, seed=2, scale=0.3)
    plan = backend.rope_plan(dim, base=500000.0)
    stream = torch.cuda.Stream()

    def buffers(rows):
        return {"rows": torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda"),
                "kv": torch.zeros(3, dtype=torch.int32, device="cuda"), "pos": torch.zeros(sum(rows), dtype=torch.int32, device="cuda"),
                "tok": torch.zeros(sum(rows), dtype=torch.int64, device="cuda"), "u": torch.zeros(3, device="cuda"),
                "qkv": torch.zeros(sum(rows), wide, device="cuda"), "out": torch.zeros(sum(rows), heads, dim, device="cuda"),
                "logits": torch.zeros(3, vocab, device="cuda"), "ids": torch.zeros(3, dtype=torch.int32, device="cuda")}

    def step(b, rows):
        s = torch.cuda.current_stream().cuda_stream
        batch = backend.paged_batch(b["rows"].data_ptr(), b["kv"].data_ptr(), p.dev[2].data_ptr(), p.width, 3, sum(rows), max(rows), 64)
        q = b["qkv"]
        q.copy_(table[b["tok"]])
        backend.dev_rope(plan, b["pos"].data_ptr(), q.data_ptr(), q.data_ptr(), sum(rows), heads + kv_heads, dim, (wide, dim), (wide, dim), F32, s)
        backend.dev_cache_write(p.cache(), batch, q[:, heads * dim :].data_ptr(), q[:, (heads + kv_heads) * dim :].data_ptr(), F32, wide, dim, s)
        a = backend.paged_attention(q.data_ptr(), b["out"].data_ptr(), F32, heads, wide, dim, heads * dim, dim, dim**-0.5)
        assert backend.paged_attention_workspace(p.cache(), batch, a) == 0
        backend.dev_paged_attention(p.cache(), batch, a, s)
        last = (b["rows"][1:] - 1).long()
        torch.matmul(b["out"][last].view(3, -1), head, out=b["logits"])
        backend.dev_sample_rows(b["logits"].data_ptr(), F32, 3, vocab, vocab, None, None, None, None, b["u"].data_ptr(), b["ids"].data_ptr(), None, s)

    rng = np.random.default_rng(0)
    tokens = [list(rng.integers(0, vocab, n)) for n in prompt]
    one = buffers([1, 1, 1])
    graph = None
    for i in range(steps + 1):
        rows = prompt if i == 0 else [1, 1, 1]
        b = buffers(rows) if i == 0 else one
        lens = [n + i for n in prompt]
        b["tok"].copy_(torch.tensor(sum(([*t[-r:]] for t, r in zip(tokens, rows)), [])))
        b["pos"].copy_(torch.tensor(np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)]), dtype=torch.int32))
        b["kv"].copy_(torch.tensor(lens, dtype=torch.int32))
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
        # the step by its definitions
        x = table.double().cpu().numpy()[np.concatenate([t[-r:] for t, r in zip(tokens, rows)])].reshape(-1, heads + 2 * kv_heads, dim)
        freq = 500000.0 ** (-2.0 * np.arange(dim // 2) / dim)
        pos = b["pos"].cpu().numpy()
        x[:, : heads + kv_heads] = turned(x[:, : heads + kv_heads], pos, freq, dim, False)
        full = (p.rows, p.kv, p.starts)
        p.rows, p.kv, p.starts = rows, lens, np.concatenate([[0], np.cumsum(rows)])
        assert np.abs(b["qkv"].double().cpu().numpy().reshape(x.shape) - x).max() <= 16 * 2.0**-24 * np.abs(x).max()
        unit = 1 / 250 if cache == I8 else 2.0**-11  # half a step of the cache's type, of the vector's largest
        for s in range(3):
            new = slice(p.starts[s], p.starts[s + 1])
            for which, at in ((0, heads), (1, heads + kv_heads)):
                rows_of = x[new, at : at + kv_heads]
                assert np.all(np.abs(p.get(which, s)[lens[s] - rows[s] :] - rows_of) <= unit * np.abs(rows_of).max(-1, keepdims=True))
        qd = b["qkv"].double().cpu().numpy().reshape(x.shape)[:, :heads]
        want, _, weight, reach = attention(p, qd, dim**-0.5, True, 0)
        bound, _ = attention_bounds(want, weight, reach, dim, max(lens), F32)
        assert np.all(np.abs(b["out"].double().cpu().numpy() - want) <= bound)
        logits = b["logits"].double().cpu().numpy()
        for s in range(3):
            want_id, _, gap = sample(logits[s], 1.0, 0, 1.0, 0.0, float(u[s]))
            assert gap <= 1e-11 or int(b["ids"][s]) == want_id
            tokens[s].append(int(b["ids"][s]))
        p.rows, p.kv, p.starts = full
