"""The serving operators' definitions in 64 bits (numpy), and the buffers that their tests share."""
import math

import numpy as np
import torch

from mimir_framework_b200 import abi, runtime as rt

TORCH = {abi.T_F32: torch.float32, abi.T_F16: torch.float16, abi.T_BF16: torch.bfloat16, abi.T_I8: torch.int8, abi.T_E4M3: torch.float8_e4m3fn}
TOP = {abi.T_I8: 127.0, abi.T_E4M3: 448.0}


def half_step(type_):
    """The largest relative error of one rounding to the type."""
    return torch.finfo(TORCH[type_]).eps / 2


class Pages:
    """A cache, a ragged batch over it and its page table in a shuffled order; unused slots and table entries hold rubbish."""

    def __init__(self, rows, kv, kv_heads, dim, page, type_, order="slot", seed=0, spare=3, gap=0):
        rng = np.random.default_rng(seed)
        self.rows, self.kv, self.heads, self.dim, self.page, self.type, self.order = list(rows), list(kv), kv_heads, dim, page, type_, order
        need = [-(-n // page) for n in kv]
        self.width = max(max(need, default=0), 1) + 1
        self.n_pages = sum(need) + spare
        free = list(rng.permutation(self.n_pages))
        self.table = np.full((len(kv), self.width), -77, np.int32)
        for i, n in enumerate(need):
            for j in range(n):
                self.table[i, j] = free.pop()
        wide = dim + gap  # of a head in the pages
        shape = (self.n_pages, page, kv_heads, wide) if order == "slot" else (self.n_pages, kv_heads, page, wide)
        self.strides = (page * kv_heads * wide, kv_heads * wide, wide) if order == "slot" else (page * kv_heads * wide, wide, page * wide)
        rubbish = torch.full(shape, float("nan"))
        self.pool = [(torch.full(shape, 99, dtype=torch.int8) if type_ == abi.T_I8 else rubbish.to(TORCH[type_])).cuda() for _ in range(2)]
        self.scale = [torch.full((self.n_pages, kv_heads, page), float("nan"), device="cuda") for _ in range(2)] if type_ in TOP else [None, None]
        self.starts = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.n_rows = int(self.starts[-1])
        self.dev = [torch.from_numpy(np.asarray(v, np.int32)).cuda() for v in (self.starts, self.kv, self.table)]

    def cache(self, **change):
        c = dict(k=self.pool[0].data_ptr(), v=self.pool[1].data_ptr(), type=self.type, n_pages=self.n_pages, page_size=self.page, kv_heads=self.heads,
                 head_dim=self.dim, page_stride=self.strides[0], slot_stride=self.strides[1], head_stride=self.strides[2],
                 k_scale=self.scale[0].data_ptr() if self.scale[0] is not None else None,
                 v_scale=self.scale[1].data_ptr() if self.scale[1] is not None else None)
        c.update(change)
        return rt.paged_cache(**c)

    def batch(self, **change):
        b = dict(row_start=self.dev[0].data_ptr(), kv_len=self.dev[1].data_ptr(), page_table=self.dev[2].data_ptr(), table_stride=self.width,
                 n_seqs=len(self.kv), n_rows=self.n_rows, max_rows=max(self.rows, default=0), max_kv=max(self.kv, default=0))
        b.update(change)
        return rt.paged_batch(**b)

    def slots(self, name, seq, keys):
        """Indices of those keys' slots in pool and scale."""
        page, slot = self.table[seq][np.asarray(keys) // self.page], np.asarray(keys) % self.page
        return page, slot

    def put(self, which, seq, keys, values):
        """Stores fp32 [keys][heads][dim] as the cache's type (numpy's and torch's roundings, not the framework's)."""
        page, slot = (torch.from_numpy(np.asarray(v, np.int64)).cuda() for v in self.slots(which, seq, keys))
        x = values.float()
        if self.type in TOP:
            scale = x.abs().amax(-1) * torch.tensor(1.0 / TOP[self.type], dtype=torch.float32, device="cuda")
            x = x / scale[..., None]
            x = x.round().to(torch.int8) if self.type == abi.T_I8 else x.to(torch.float8_e4m3fn)
            self.scale[which][page, :, slot] = scale
        x = x.to(self.pool[which].dtype)
        pool = self.pool[which]
        if self.type == abi.T_E4M3:
            x, pool = x.view(torch.uint8), pool.view(torch.uint8)
        if self.order == "slot":
            pool[page, slot, :, : self.dim] = x
        else:
            pool[page, :, slot, : self.dim] = x

    def get(self, which, seq):
        """What the cache holds for a sequence, in 64 bits: [keys][heads][dim]."""
        keys = np.arange(self.kv[seq])
        page, slot = (torch.from_numpy(np.asarray(v, np.int64)).cuda() for v in self.slots(which, seq, keys))
        pool = self.pool[which]
        x = (pool.float()[page, slot] if self.order == "slot" else pool.float()[page, :, slot])[..., : self.dim].double()
        if self.type in TOP:
            x = x * self.scale[which][page, :, slot].double()[..., None]
        return x.cpu().numpy()

    def fill(self, seed=1, spread=1.0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        for which in range(2):
            for s, n in enumerate(self.kv):
                self.put(which, s, np.arange(n), torch.randn(n, self.heads, self.dim, generator=g, device="cuda") * spread)


def attention(pages, q, scale, causal, window):
    """out, lse, and for each output the sum of p |v| and the largest |q| |k| scale of its row's keys (for error bounds)."""
    rows, heads, dim = q.shape
    group = heads // pages.heads
    out, lse, weight, reach = (np.zeros((rows, heads, dim)), np.full((rows, heads), -np.inf), np.zeros((rows, heads, dim)), np.zeros((rows, heads, 1)))
    for s, (n_new, n) in enumerate(zip(pages.rows, pages.kv)):
        if not n_new or not n:
            continue
        k, v = pages.get(0, s), pages.get(1, s)
        a = pages.starts[s]
        pos = n - n_new + np.arange(n_new)
        key = np.arange(n)
        seen = np.ones((n_new, n), bool)
        if causal:
            seen &= key[None] <= pos[:, None]
        if window:
            seen &= key[None] > pos[:, None] - window
        for h in range(heads):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[a : a + n_new, h]
            z = np.where(seen, qq @ kk.T * scale, -np.inf)
            top = z.max(1, keepdims=True)
            with np.errstate(invalid="ignore", divide="ignore"):
                e = np.where(seen, np.exp(z - np.where(np.isfinite(top), top, 0.0)), 0.0)
                total = e.sum(1, keepdims=True)
                p = np.where(total > 0, e / total, 0.0)
                lse[a : a + n_new, h] = np.where(total > 0, top + np.log(total), -np.inf)[:, 0]
            out[a : a + n_new, h] = p @ vv
            weight[a : a + n_new, h] = p @ np.abs(vv)
            reach[a : a + n_new, h] = np.where(seen, np.abs(qq) @ np.abs(kk).T, 0.0).max(1, keepdims=True) * abs(scale)
    return out, lse, weight, reach


def attention_bounds(out, weight, reach, dim, keys, type_, chunk=False, one_half=False):
    """How far a result may be: |d out| and |d lse|.

    Score: a term of 22 bits a factor (2^-22 each of two), head_dim / 16 steps of up to three tensor instructions whose truncating sums
    lose up to 2^-22 of the terms' magnitudes each, the scale and the exponent's base (2^-23), exp2 (2 units, 2^-22 of p).
    Values: probabilities of 22 bits (2^-22), six instructions a block of keys (6 * 2^-22), the running sums' fp32 additions, one
    for each block of 16 keys of a warp and each of up to 64 parts that meet (2^-24 each), the sum of probabilities likewise, the division.
    The result's type rounds once.  bfloat16 probabilities are hi + lo, 16 bits: 2^-17.  In chunks of many rows of 16 bits (`chunk`) a
    probability is one number of the cache's 16-bit type (half for 8-bit caches): it is off by half a step of its own, and so is each p |v|.
    So is it by half's, 2^-11, where a bfloat16 result comes from a cache of half or 8 bits (`one_half`).  There a bfloat16 query may become a half times its row's largest: 2^-25 of that, less than the terms' 2^-21 of the reach."""
    score = reach * (2.0**-21 + 3 * math.ceil(dim / 16) * 2.0**-22 + 2.0**-23) * 1.5
    sums = (keys / 16 + 80) * 2.0**-24
    value = (2.0**-17 if type_ == abi.T_BF16 else 2.0**-22) + 6 * 2.0**-22 + 2.0**-21
    if chunk:
        value += half_step(type_)
    if one_half:
        value += 2.0**-11
    inner = weight * (2 * score + 2 * sums + value)
    return inner + (np.abs(out) + inner) * half_step(type_) + (2.0**-24 if type_ == abi.T_F16 else 0.0), score[..., 0] + sums + 2.0**-21


def sample(x, t, k, p, m, u):
    """(index, logarithm of its share, distance of u from the nearest border) of one row of 64-bit logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    if not (x > -np.inf).any():
        return -1, -np.inf, 1.0
    order = np.argsort(-x, kind="stable")
    if x[order[0]] == np.inf or not t > 0:
        return int(order[0]), 0.0, 1.0
    order = order[x[order] > -np.inf]
    if 0 < k < len(x):
        order = order[:k]
    w = np.exp((x[order] - x[order[0]]) / float(t))
    if p < 1:
        order = order[: max(1, int(np.sum(np.cumsum(w) - w < float(p) * w.sum())))]
    w = np.exp((x[order] - x[order[0]]) / float(t))
    order = order[w >= min(float(m), 1.0)]
    order = np.sort(order)
    w = np.exp((x[order] - x.max()) / float(t))
    run = np.cumsum(w)
    i = min(int(np.sum(run <= float(u) * run[-1])), len(order) - 1)
    return int(order[i]), float(np.log(w[i] / run[-1])), float(np.abs(run / run[-1] - float(u)).min())
