"""Serving calls at the ends of what they accept."""
import math
import threading
import time

import numpy as np
import pytest
import torch

from mimir_framework_b200 import abi
from serving_ref import TORCH, Pages, attention, attention_bounds, sample

pytestmark = pytest.mark.gpu
F32, F16, BF16, I8, E4M3 = abi.T_F32, abi.T_F16, abi.T_BF16, abi.T_I8, abi.T_E4M3


def normal(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def attend(backend, p, q, type_, scale, causal=True, window=0, **batch):
    """out and lse of q [rows][heads][dim] over the pages."""
    rows, heads, dim = q.shape
    out, lse = torch.full_like(q, -7.0), torch.full((rows, heads), -7.0, device="cuda")
    b = p.batch(**batch)
    a = backend.paged_attention(q.data_ptr(), out.data_ptr(), type_, heads, heads * dim, dim, heads * dim, dim, scale, causal, window, lse.data_ptr())
    size = backend.paged_attention_workspace(p.cache(), b, a)
    ws = torch.full((size + 16,), 255, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    backend.dev_paged_attention(p.cache(), b, a)
    torch.cuda.synchronize()
    backend.check_device()
    return out, lse


def held(p, q, out, lse, type_, scale, causal, window, chunk):
    want, want_lse, weight, reach = attention(p, q.double().cpu().numpy(), scale, causal, window)
    bound, lse_bound = attention_bounds(want, weight, reach, p.dim, max(p.kv), BF16 if p.type == BF16 else type_, chunk and type_ != F32,
                                        type_ == BF16 and p.type != BF16)
    err = np.abs(out.double().cpu().numpy() - want)
    assert np.all(err <= bound), f"{np.max(err / np.maximum(bound, 1e-300))} of the bound"
    got, some = lse.double().cpu().numpy(), ~np.isneginf(want_lse)
    assert np.array_equal(~np.isneginf(got), some)
    got, want_lse, lse_bound = got[some], want_lse[some], lse_bound[some]
    assert np.all(np.abs(got - want_lse) <= lse_bound + np.abs(want_lse) * 2.0**-22)


# ---- scores --------------------------------------------------------------------------------------------------------------------------
PAIRS = [(BF16, BF16), (F16, F16), (F16, BF16), (F16, F32), (I8, F16), (I8, BF16), (I8, F32), (E4M3, F16), (E4M3, BF16), (E4M3, F32), (F32, F32)]


@pytest.mark.parametrize("cache,type_", PAIRS)
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-30, -1e-30])
@pytest.mark.parametrize("rows,kv,dim,causal,window", [([150, 3], [400, 130], 64, True, 0), ([140, 70], [300, 50], 64, True, 33), ([160], [333], 128, False, 0)])
def test_a_scale_of_zero_or_next_to_it_is_the_mean(backend, rows, kv, dim, causal, window, scale, cache, type_):
    """Many rows and few; some queries are all zeros, whose products vanish with the scale."""
    p = Pages(rows, kv, 1, dim, 16, cache, seed=dim)
    p.fill()
    q = normal(p.n_rows, 2, dim, seed=3, dtype=TORCH[type_])
    q[::5] = 0.0
    out, lse = attend(backend, p, q, type_, scale, causal, window)
    held(p, q, out, lse, type_, scale, causal, window, True)


@pytest.mark.parametrize("cache,type_", [(BF16, BF16), (F16, F16), (F16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("rows,causal", [(150, False), (150, True), (2, False)])
@pytest.mark.parametrize("at", [0, 6, 7, 14, 29, 127])
def test_a_key_that_is_no_number_makes_every_row_that_sees_it_none(backend, rows, causal, at, cache, type_):
    """In any column of a tile without masks and in one with them; rows before it and other heads go on."""
    kv = 384
    p = Pages([rows], [kv], 2, 64, 16, cache, seed=2)
    p.fill()
    q = normal(rows, 4, 64, seed=3, dtype=TORCH[type_])
    clean, clean_lse = attend(backend, p, q, type_, 0.125, causal)
    held(p, q, clean, clean_lse, type_, 0.125, causal, 0, True)
    for key in (at, 256 + at):
        page, slot = p.slots(0, 0, [key])
        where = (int(page[0]), int(slot[0]), 1)
        kept = p.pool[0][where].clone()
        p.pool[0][where] = float("nan")
        out, lse = attend(backend, p, q, type_, 0.125, causal)
        p.pool[0][where] = kept
        sees = torch.arange(kv - rows, kv, device="cuda") >= key if causal else torch.ones(rows, dtype=torch.bool, device="cuda")
        assert out[sees][:, 2:].isnan().all() and lse[sees][:, 2:].isnan().all()
        out[sees, 2:], lse[sees, 2:] = clean[sees, 2:], clean_lse[sees, 2:]
        held(p, q, out, lse, type_, 0.125, causal, 0, True)


# ---- sampling ----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,top_p,min_p,type_", [("many small", 0.998, 0.0015, F32), ("many small", 0.998, 0.0015, BF16), ("equals", 0.995, 0.5, BF16), ("equals", 0.6, 0.5, F16)])
def test_sampling_by_mass_and_least_share_of_the_most_logits(backend, kind, top_p, min_p, type_):
    """Shares that are less than a rough sum resolves, or all off the same way."""
    n = 1 << 24
    if kind == "many small":  # a quarter at one, the rest at about two thousandths
        x = torch.full((1, n), -6.25, device="cuda")
        x[:, ::4] = 0.0
    else:  # each one's share is nearly half a unit of 2^-30 off
        x = torch.zeros(1, n, device="cuda")
        x[:, : n - round(2**30 / 66.49)] = -float("inf")
    x = x.to(TORCH[type_])
    u, p, m = (torch.full((1,), v, device="cuda") for v in (0.5 if kind == "many small" else 0.9999, top_p, min_p))
    ids, logp = torch.full((1,), -7, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda")
    backend.dev_sample_rows(x.data_ptr(), type_, 1, n, n, None, None, p.data_ptr(), m.data_ptr(), u.data_ptr(), ids.data_ptr(), logp.data_ptr())
    torch.cuda.synchronize()
    want, lp, _ = sample(x[0].double().cpu().numpy(), 1.0, 0, float(p[0]), float(m[0]), float(u[0]))
    # the reference adds 2^24 numbers up one after the other: off by up to 2^-29 of 2^22 or so, which is four of the small ones
    assert abs(int(ids[0]) - want) <= (5 if kind == "many small" else 0)
    assert abs(float(logp[0]) - lp) <= 2.0**-22 * max(1.0, abs(lp))


@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (0, 1.0 - 2.0**-20), (3000, 1.0), (200, 1.0), (900, 1.0)])
@pytest.mark.parametrize("down", [3.0, 15.0, 22.0, 27.0, 30.0])
def test_the_logarithm_of_a_small_share_keeps_its_bits(backend, down, top_k, top_p):
    """The first index is taken (uniform 0), whose share is e^-down or less."""
    n = 70000
    x = normal(2, n, seed=4, scale=1.0) - 45.0
    x[:, 0] = -down + 0.123
    x[1, : top_k // 2] = -down + 0.123
    x[:, 7000:7100] = normal(2, 100, seed=5, scale=0.1).clamp(max=0.4)
    x[:, 7050] = 0.5
    u, k, p = torch.zeros(2, device="cuda"), torch.full((2,), top_k, dtype=torch.int32, device="cuda"), torch.full((2,), top_p, device="cuda")
    ids, logp = torch.full((2,), -7, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    backend.dev_sample_rows(x.data_ptr(), F32, 2, n, n, None, k.data_ptr(), p.data_ptr(), None, u.data_ptr(), ids.data_ptr(), logp.data_ptr())
    torch.cuda.synchronize()
    for r in range(2):
        want, lp, _ = sample(x[r].double().cpu().numpy(), 1.0, top_k, float(p[r]), 0.0, 0.0)
        # two logarithms of fp32 that do not cancel, their difference, and a sum's rounding: under four units of 2^-24 of it; a share over one half is not among them
        assert int(ids[r]) == want and abs(float(logp[r]) - lp) <= 2.0**-22 * abs(lp), (float(logp[r]), lp)


# ---- values -------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,kv,dim,group", [([1, 2], [33, 300], 64, 4), ([40], [170], 128, 2), ([3, 17], [90, 20], 256, 1), ([1], [5], 8, 1)])
@pytest.mark.parametrize("size", [1e6, 1e-3, 1e-6, 1e-20, "mixed"])
def test_fp32_caches_of_any_size(backend, size, rows, kv, dim, group):
    """Keys and values of an fp32 cache keep their bits whatever they are near, each by itself."""
    p = Pages(rows, kv, 2, dim, 8, F32, seed=4)
    p.fill()
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    for which in range(2):
        if size == "mixed":  # values over 2^60, keys over 2^20, from element to element
            span = 30.0 if which else 10.0
            f = torch.exp2(torch.rand(p.pool[which].shape, generator=g, device="cuda") * 2 * span - span)
        else:
            f = size
        p.pool[which].mul_(f)
    scale = 2.0**-8 if size == "mixed" else 1 / (size * math.sqrt(dim))
    q = normal(p.n_rows, 2 * group, dim, seed=3)
    out, lse = attend(backend, p, q, F32, scale)
    held(p, q, out, lse, F32, scale, True, 0, False)


@pytest.mark.parametrize("cache", [F16, I8, E4M3])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lead", [40.0, 12.0])
@pytest.mark.parametrize("first", [0, 64, 8064, 16320])
def test_fp32_results_of_chunks_do_not_drift_with_the_keys(backend, first, lead, dim, cache):
    """Nearly all of the probability on 64 of 16 K keys, at the beginning, in the middle or at the end.  80 sequences share the pages, so that
    none of them is divided among blocks."""
    n, rows, seqs = 16384, 40, 80
    p = Pages([rows], [n], 1, dim, 64, cache, seed=1)
    keys = torch.zeros(n, 1, dim, device="cuda")
    keys[first : first + 64, :, 0] = lead
    p.put(0, 0, np.arange(n), torch.where(keys == 0, 1e-30, keys) if cache in (I8, E4M3) else keys)
    values = normal(n, 1, dim, seed=2).abs() + 0.5  # (of one sign: nothing cancels)
    p.put(1, 0, np.arange(n), values)
    q = torch.zeros(rows, 1, dim, device="cuda")
    q[..., 0] = 1.0
    many = q.repeat(seqs, 1, 1)
    starts = torch.arange(0, rows * seqs + 1, rows, dtype=torch.int32, device="cuda")
    lens, table = p.dev[1].repeat(seqs), p.dev[2].repeat(seqs, 1).contiguous()
    out, lse = attend(backend, p, many, F32, 1.0, False, row_start=starts.data_ptr(), kv_len=lens.data_ptr(), page_table=table.data_ptr(), n_seqs=seqs,
                      n_rows=rows * seqs, max_rows=rows)
    assert torch.equal(out, out[:1].expand_as(out)) and torch.equal(lse, lse[:1].expand_as(lse))
    want, want_lse, weight, _ = attention(p, q.double().cpu().numpy(), 1.0, False, 0)
    # The 64 keys' scores are one product each and alike, so what they are off by cancels.  A probability is two halves (2^-22).  The sum of
    # probabilities has half a unit (2^-24) each of up to 96 additions within a tile, and sum and products one for each tile added to them, where
    # the others' probabilities are not zero (64 and 128 keys do not meet a border: one tile has nearly all).  Two tiles' products are 32 instructions
    # that truncate, by a unit (2^-23) at most.  The others' share is under 1e-3, and their scores' 2^-21 * 12 count for that.
    tiles = 128 if lead < 20 else 1
    bound = 2.0**-22 + (96 + 2 * tiles) * 2.0**-24 + 32 * 2.0**-23 + 12 * 2.0**-21 * 1e-3 + 2.0**-23
    err = np.abs(out[:rows].double().cpu().numpy() - want)
    assert np.all(err <= bound * weight), f"{np.max(err / weight)}, bound {bound}"


@pytest.mark.parametrize("cache,type_,few", [(BF16, BF16, 32), (F16, F16, 32), (F16, BF16, 32), (F16, F32, 32), (I8, F16, 64), (I8, BF16, 64), (E4M3, F16, 64), (E4M3, F32, 32)])
@pytest.mark.parametrize("dim,window", [(64, 0), (128, 90)])
def test_few_rows_beside_chunks_keep_their_terms(backend, dim, window, cache, type_, few):
    """A sequence of few rows is as exact in a batch with chunks as alone: its probabilities have two terms."""
    rows, kv = [200, 1, few, few - 3, 150], [300, 777, 100, few - 9, 400]
    p = Pages(rows, kv, 2, dim, 16, cache, seed=5)
    p.fill()
    q = normal(p.n_rows, 2, dim, seed=3, dtype=TORCH[type_])
    out, lse = attend(backend, p, q, type_, dim**-0.5, True, window)
    held(p, q, out, lse, type_, dim**-0.5, True, window, True)
    want, _, weight, reach = attention(p, q.double().cpu().numpy(), dim**-0.5, True, window)
    bound, _ = attention_bounds(want, weight, reach, dim, max(kv), BF16 if cache == BF16 else type_, False, type_ == BF16 and cache != BF16)
    err = np.abs(out.double().cpu().numpy() - want)
    for s in (1, 2, 3):
        at = slice(p.starts[s], p.starts[s + 1])
        assert np.all(err[at] <= bound[at]), f"{np.max(err[at] / np.maximum(bound[at], 1e-300))} of the bound"


# ---- findings ------------------------------------------------------------------------------------------------------------------------------
def test_findings_are_reported_once_whoever_asks(backend):
    """One thread makes bad calls of changing kinds and asks after each; another asks all the time, of another stream.  Every finding reaches one
    of them, and is gone then."""
    p = Pages([1], [40], 1, 64, 16, F16, seed=9)
    p.fill()
    x = normal(1, 1, 64, dtype=torch.float16)
    bad_rows, bad_len = torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.tensor([99], dtype=torch.int32, device="cuda")
    bad_page = torch.full_like(p.dev[2], -1)
    torch.cuda.synchronize()
    kinds = [("row ranges", p.batch(row_start=bad_rows.data_ptr())), ("key count", p.batch(kv_len=bad_len.data_ptr())), ("page number", p.batch(page_table=bad_page.data_ptr()))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    seen, rounds, stop, trouble = [], [0], threading.Event(), []

    def ask(stream):
        try:
            backend.check_device(stream.cuda_stream)
        except backend.MimirB200Error as e:
            seen.append(str(e))

    def other():
        try:
            torch.cuda.set_device(0)
            while not stop.is_set():
                ask(streams[1])
                rounds[0] += 1
        except Exception as e:  # (the first thread must not wait for good)
            trouble.append(e)

    thread = threading.Thread(target=other)
    thread.start()
    lost = []
    try:
        for i in range(999):
            what, batch = kinds[i % 3]
            before = len(seen)
            backend.dev_cache_write(p.cache(), batch, x.data_ptr(), x.data_ptr(), F16, 64, 64, streams[0].cuda_stream)
            ask(streams[0])
            now = rounds[0]
            # (a finding that the other has taken it has told two rounds later)
            while not any(what in s for s in seen[before:]) and rounds[0] < now + 2 and not trouble:
                time.sleep(0)
            if not any(what in s for s in seen[before:]):
                lost.append(i)
    finally:
        stop.set()
        thread.join()
    assert not trouble and not lost, (trouble, len(lost))
    assert [sum(what in s for s in seen) for what, _ in kinds] == [333, 333, 333]
