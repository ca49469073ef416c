"""Cases of the serving operators on a paged key / value cache: rotary positions, writing the cache (whole or in 8 bits), reading it
back, attention of new tokens over it, and choosing a token from logits.

``run`` computes them in plain torch operations, or, with ``own`` set, through the framework's device-pointer calls.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODES = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3, "e4m3": 4}  # of the framework's calls
TOP = {"i8": 127.0, "e4m3": 448.0}  # largest code


def listed():
    return [
        # one generated token for each of 32 conversations: queries and keys of one layer, side by side
        dict(name="rope step", op="rope", rows=32, heads=40, dim=128, rot=128, inter=False, type="bf16", scaling="none", far=100000),
        # a prompt's queries and keys in the framework's own type, half of each head turned, context stretched
        dict(name="rope prompt", op="rope", rows=8192, heads=40, dim=128, rot=64, inter=True, type="f32", scaling="ramp", far=131072),
        # one new token of each of 64 conversations stored in 8-bit floats
        dict(name="write step", op="write", seqs=64, new=1, ctx=1024, kv_heads=8, dim=128, page=16, cache="e4m3", type="bf16", order="slot"),
        # chunks of several prompts stored as 8-bit integers, ragged
        dict(name="write prompts", op="write", seqs=8, new=4096, ctx=6000, kv_heads=8, dim=128, page=64, cache="i8", type="bf16", order="head"),
        # a few sequences of odd lengths fetched from the cache in the framework's own type
        dict(name="read few", op="read", seqs=3, new=1, ctx=333, kv_heads=12, dim=64, page=16, cache="e4m3", type="f32", order="slot"),
        # sequences moved out of an 8-bit cache
        dict(name="read many", op="read", seqs=16, new=1, ctx=8192, kv_heads=8, dim=128, page=64, cache="i8", type="bf16", order="slot"),
        # one token of one conversation with the framework's decoder: 12 heads of 64 in fp32
        dict(name="attention one token", op="attention", seqs=1, new=1, ctx=1024, heads=12, kv_heads=12, dim=64, page=16, cache="f16", type="f32",
             order="slot", causal=True, window=0),
        # a batch of conversations of different lengths, one token each, grouped heads
        dict(name="attention batch step", op="attention", seqs=64, new=1, ctx=4096, heads=32, kv_heads=8, dim=128, page=16, cache="bf16", type="bf16",
             order="slot", causal=True, window=0),
        # a few very long documents in an 8-bit cache
        dict(name="attention long step", op="attention", seqs=4, new=1, ctx=131072, heads=32, kv_heads=8, dim=128, page=64, cache="e4m3", type="bf16",
             order="head", causal=True, window=0),
        # chunks of new tokens of several prompts behind what is cached already, ragged
        dict(name="attention chunks", op="attention", seqs=4, new=2048, ctx=8192, heads=32, kv_heads=8, dim=128, page=64, cache="bf16", type="bf16",
             order="slot", causal=True, window=0),
        # the next token of one conversation, vocabulary of the framework's decoder
        dict(name="sample one", op="sample", rows=1, n=32000, type="f32", top_k=50, top_p=0.9, min_p=0.0, spread=3.0),
        # the next tokens of a large batch over a large vocabulary, every filter on
        dict(name="sample batch", op="sample", rows=256, n=128256, type="bf16", top_k=0, top_p=0.95, min_p=0.02, spread=3.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attention", "attention", "attention", "sample"])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        heads = rng.randint(1, 48)
        rows = _log(rng, 1, max(1, 41_000_000 // (heads * dim)))
        return dict(op=op, rows=rows, heads=heads, dim=dim, rot=rot, inter=rng.random() < 0.5, type=rng.choice(["f32", "f16", "bf16"]),
                    scaling=rng.choice(["none", "linear", "bands", "ramp"]), far=rng.choice([4000, 131072, 2000000]))
    if op == "sample":
        n = _log(rng, 100, 200000)
        return dict(op=op, rows=_log(rng, 1, min(1024, 32_000_000 // n)), n=n, type=rng.choice(["f32", "f16", "bf16"]), top_k=rng.choice([0, 0, 1, 40, 1000]),
                    top_p=rng.choice([1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.05]), spread=rng.choice([0.5, 2.0, 4.0]))
    cache = rng.choice(["f32", "f16", "bf16", "i8", "e4m3"])
    kind = {"f32": ["f32"], "f16": ["f16", "f32"], "bf16": ["bf16"]}.get(cache, ["f32", "f16", "bf16"])
    case = dict(op=op, kv_heads=rng.randint(1, 8), dim=rng.choice([32, 64, 80, 96, 128, 128, 192, 256]), page=rng.choice([8, 16, 16, 24, 32, 64, 128]), cache=cache,
                type=rng.choice(kind if op == "attention" else ["f32", "f16", "bf16"]), order=rng.choice(["slot", "head"]))
    wide = case["kv_heads"] * case["dim"]
    if op != "attention":
        case |= dict(seqs=_log(rng, 1, 128), ctx=_log(rng, 1, 16384), new=1)
        case["ctx"] = max(1, min(case["ctx"], 60_000_000 // (case["seqs"] * wide)))
        if op == "write":
            case["new"] = _log(rng, 1, case["ctx"])
        return case
    case |= dict(heads=case["kv_heads"] * rng.choice([1, 2, 4, 5, 8]), causal=rng.random() < 0.8, window=rng.choice([0, 0, 0, 100, 1000]))
    if rng.random() < 0.5:
        case |= dict(seqs=_log(rng, 1, 128), new=rng.choice([1, 1, 1, 2, 5]), ctx=_log(rng, 8, 65536))
        case["ctx"] = max(8, min(case["ctx"], 120_000_000 // (case["seqs"] * wide)))
    else:
        case |= dict(seqs=_log(rng, 1, 8), new=_log(rng, 16, 2048), ctx=_log(rng, 16, 8192))
        case["ctx"] = max(case["ctx"], case["new"])
        case["ctx"] = min(case["ctx"], 150_000_000_000 // (case["seqs"] * case["new"] * case["heads"] * case["dim"]))
        case["new"] = min(case["new"], case["ctx"])
    return case


def _lengths(case):
    """New rows and keys of each sequence: the first has the most of both, the others between a half and all."""
    r = np.random.RandomState(case["ctx"])
    n = case["seqs"]
    kv = np.maximum(1, (case["ctx"] * r.uniform(0.5, 1.0, n))).astype(np.int64)
    new = np.maximum(1, np.round(case["new"] * r.uniform(0.5, 1.0, n))).astype(np.int64)
    kv[0], new[0] = case["ctx"], case["new"]
    return np.minimum(new, kv), kv


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "rope":
        s["x"] = normal(case["rows"], case["heads"], case["dim"], dtype=TYPES[case["type"]])
        s["pos"] = torch.randint(0, case["far"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        s["y"] = torch.empty_like(s["x"])
    elif case["op"] == "sample":
        rows = case["rows"]
        s["x"] = normal(rows, case["n"], scale=case["spread"], dtype=TYPES[case["type"]])
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        s["t"] = 0.5 + torch.rand(rows, generator=g, device="cuda")
        s["t"][rows - 1 :: 17] = 0.0 if rows > 1 else 0.8  # some users want the likeliest token
        s["k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
        s["p"] = torch.full((rows,), case["top_p"], device="cuda")
        s["m"] = torch.full((rows,), case["min_p"], device="cuda")
        s["ids"], s["logp"] = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    else:
        new, kv = _lengths(case)
        page, heads, dim, kind = case["page"], case["kv_heads"], case["dim"], case["cache"]
        need = (kv + page - 1) // page
        width, total = int(need.max()), int(need.sum())
        pages = total + 3
        table = np.zeros((len(kv), width), np.int32)
        order = np.random.RandomState(seed % (1 << 31)).permutation(pages)[:total].astype(np.int32)
        ends = np.cumsum(need)
        for i, n in enumerate(need):
            table[i, :n] = order[ends[i] - n : ends[i]]
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        rows = int(starts[-1])
        s |= {"rows": rows, "new": int(new.max()), "kv": int(kv.max()), "pages": pages, "width": width}
        s["starts"], s["kv_len"], s["table"] = (torch.from_numpy(v).cuda() for v in (starts, kv.astype(np.int32), table))
        shape = (pages, page, heads, dim) if case["order"] == "slot" else (pages, heads, page, dim)
        for name in ("k", "v"):
            if case["op"] == "write":
                pool = torch.zeros(shape, dtype=torch.int8 if kind == "i8" else torch.float32, device="cuda").to(TYPES[kind])
            elif kind == "i8":
                pool = normal(*shape, scale=40.0).clamp_(-127, 127).to(torch.int8)
            else:
                pool = normal(*shape, scale=100.0 if kind == "e4m3" else 1.0)
                pool = (pool.clamp_(-TOP[kind], TOP[kind]) if kind in TOP else pool).to(TYPES[kind])
            s["pool_" + name] = pool
            if kind in TOP:
                s["scale_" + name] = (torch.rand(pages, heads, page, generator=g, device="cuda") + 0.5) * (4.0 / TOP[kind]) * float(case["op"] != "write")
        t = TYPES[case["type"]]
        if case["op"] == "write":
            s["k"], s["v"] = normal(rows, heads, dim, dtype=t), normal(rows, heads, dim, dtype=t)
        elif case["op"] == "read":
            s["out_starts"] = torch.from_numpy(np.concatenate([[0], np.cumsum(kv)]).astype(np.int32)).cuda()
            s["out_rows"] = int(kv.sum())
            s["k"], s["v"] = (torch.empty(s["out_rows"], heads, dim, dtype=t, device="cuda") for _ in range(2))
        else:
            s["q"] = normal(rows, case["heads"], dim, dtype=t)
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(rows, case["heads"], device="cuda")
            s["scale"] = 1.0 / math.sqrt(dim)
    if own:
        s["own"] = _own_plan(case, s)
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------------


def _rope_spec(case):
    base = dict(rot_dim=case["rot"], base=10000.0, interleaved=case["inter"])
    if case["scaling"] == "linear":
        base |= dict(scaling="linear", factor=4.0)
    elif case["scaling"] == "bands":
        base |= dict(scaling="bands", factor=8.0, low=1.0, high=4.0, original_len=8192)
    elif case["scaling"] == "ramp":
        base |= dict(scaling="ramp", factor=16.0, low=1.0, high=32.0, original_len=8192, magnitude=0.1 * math.log(16.0) + 1.0)
    return base


def _own_plan(case, s):
    """What a program keeps: the descriptions of its buffers, and a workspace."""
    from mimir_framework_b200 import runtime as rt

    rt.init(0)
    if case["op"] == "rope":
        return rt.rope_plan(**_rope_spec(case))
    if case["op"] == "sample":
        return None
    slot, head = (case["kv_heads"] * case["dim"], case["dim"]) if case["order"] == "slot" else (case["dim"], case["page"] * case["dim"])
    cache = rt.paged_cache(k=s["pool_k"].data_ptr(), v=s["pool_v"].data_ptr(), type=CODES[case["cache"]], n_pages=s["pages"], page_size=case["page"],
                           kv_heads=case["kv_heads"], head_dim=case["dim"], page_stride=case["page"] * case["kv_heads"] * case["dim"], slot_stride=slot,
                           head_stride=head, k_scale=s["scale_k"].data_ptr() if "scale_k" in s else None,
                           v_scale=s["scale_v"].data_ptr() if "scale_v" in s else None)
    batch = rt.paged_batch(row_start=s["starts"].data_ptr(), kv_len=s["kv_len"].data_ptr(), page_table=s["table"].data_ptr(), table_stride=s["width"],
                           n_seqs=case["seqs"], n_rows=s["rows"], max_rows=s["new"], max_kv=s["kv"])
    if case["op"] != "attention":
        return cache, batch
    att = rt.paged_attention(q=s["q"].data_ptr(), out=s["out"].data_ptr(), lse=s["lse"].data_ptr(), type=CODES[case["type"]], heads=case["heads"],
                             row_stride=case["heads"] * case["dim"], head_stride=case["dim"], out_row_stride=case["heads"] * case["dim"],
                             out_head_stride=case["dim"], scale=s["scale"], causal=case["causal"], window=case["window"])
    size = rt.paged_attention_workspace(cache, batch, att)
    if size:
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        att.workspace, att.workspace_bytes = s["workspace"].data_ptr(), size
    return cache, batch, att


def _run_own(case, s):
    from mimir_framework_b200 import runtime as rt

    stream, op = torch.cuda.current_stream().cuda_stream, case["op"]
    if op == "rope":
        strides = (case["heads"] * case["dim"], case["dim"])
        rt.dev_rope(s["own"], s["pos"].data_ptr(), s["x"].data_ptr(), s["y"].data_ptr(), case["rows"], case["heads"], case["dim"], strides, strides,
                    CODES[case["type"]], stream)
        return s["y"]
    if op == "sample":
        rt.dev_sample_rows(s["x"].data_ptr(), CODES[case["type"]], case["rows"], case["n"], case["n"], s["t"].data_ptr(), s["k"].data_ptr(),
                           s["p"].data_ptr(), s["m"].data_ptr(), s["u"].data_ptr(), s["ids"].data_ptr(), s["logp"].data_ptr(), stream)
        return {"ids": s["ids"], "logp": s["logp"]}
    wide = case["kv_heads"] * case["dim"]
    if op == "write":
        cache, batch = s["own"]
        rt.dev_cache_write(cache, batch, s["k"].data_ptr(), s["v"].data_ptr(), CODES[case["type"]], wide, case["dim"], stream)
        return _pools(s)
    if op == "read":
        cache, batch = s["own"]
        rt.dev_cache_read(cache, batch, s["out_starts"].data_ptr(), s["out_rows"], s["k"].data_ptr(), s["v"].data_ptr(), CODES[case["type"]], wide,
                          case["dim"], stream)
        return {"k": s["k"], "v": s["v"]}
    cache, batch, att = s["own"]
    rt.dev_paged_attention(cache, batch, att, stream)
    return {"out": s["out"], "lse": s["lse"]}


def _pools(s):
    return {name: s[name] for name in ("pool_k", "pool_v", "scale_k", "scale_v") if name in s}


# ---- the plain forms --------------------------------------------------------------------------------------------------------


def _frequencies(case):
    """Radians a position, in 64 bits, and what cosines and sines are multiplied by."""
    rot, spec = case["rot"], _rope_spec(case)
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = 10000.0 ** (-2.0 * i / rot)
    kind = spec.get("scaling")
    if kind == "linear":
        f = f / spec["factor"]
    elif kind == "bands":
        turns = spec["original_len"] * f / (2 * math.pi)
        part = ((turns - spec["low"]) / (spec["high"] - spec["low"])).clamp(0, 1)
        f = f * (part + (1 - part) / spec["factor"])
    elif kind == "ramp":
        at = [rot * math.log(spec["original_len"] / (2 * math.pi * r)) / (2 * math.log(10000.0)) for r in (spec["high"], spec["low"])]
        first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((i - first) / (last - first if last > first else 0.001)).clamp(0, 1)
        f = f * ((1 - ramp) + ramp / spec["factor"])
    return f, spec.get("magnitude", 1.0)


def _run_rope(case, s):
    f, m = _frequencies(case)
    angle = s["pos"].double()[:, None] * f
    c, n = ((t * m).float()[:, None, :] for t in (angle.cos(), angle.sin()))
    rot, x = case["rot"], s["x"].float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["inter"] else (x[..., : rot // 2], x[..., rot // 2 : rot])
    y = torch.empty_like(x)
    u, v = a * c - b * n, a * n + b * c
    if case["inter"]:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
    else:
        y[..., : rot // 2], y[..., rot // 2 : rot] = u, v
    y[..., rot:] = x[..., rot:]
    return y.to(s["x"].dtype)


def _run_write(case, s):
    starts, kv_len = s["starts"].long(), s["kv_len"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    pos = kv_len[seq] - (starts[seq + 1] - row)
    page, slot = s["table"].long()[seq, pos // case["page"]], pos % case["page"]
    for name in ("k", "v"):
        x, pool = s[name].float(), s["pool_" + name]
        if case["cache"] in TOP:
            scale = x.abs().amax(-1) / TOP[case["cache"]]
            x = torch.where(scale[..., None] > 0, x / scale[..., None], 0.0)
            x = x.round().to(torch.int8) if case["cache"] == "i8" else x.to(torch.float8_e4m3fn)
            s["scale_" + name][page, :, slot] = scale
        x = x.to(pool.dtype)
        if case["cache"] == "e4m3":
            x, pool = x.view(torch.uint8), pool.view(torch.uint8)
        if case["order"] == "slot":
            pool[page, slot] = x
        else:
            pool[page, :, slot] = x
    return _pools(s)


def _gather(case, s, name, seq, pos):
    """fp32 keys or values at those positions of those sequences, [..., heads, dim]."""
    page, slot = s["table"].long()[seq, pos // case["page"]], pos % case["page"]
    pool = s["pool_" + name]
    x = (pool[page, slot] if case["order"] == "slot" else pool[page, :, slot]).float()
    return x * s["scale_" + name][page, :, slot][..., None] if case["cache"] in TOP else x


def _run_read(case, s):
    row = torch.arange(s["out_rows"], device="cuda")
    seq = torch.searchsorted(s["out_starts"].long(), row, right=True) - 1
    pos = row - s["out_starts"].long()[seq]
    return {name: _gather(case, s, name, seq, pos).to(TYPES[case["type"]]) for name in ("k", "v")}


def _run_attention(case, s):
    starts, kv_len = s["starts"].long(), s["kv_len"].long()
    n, most, keys, heads, dim = case["seqs"], s["new"], s["kv"], case["kv_heads"], case["dim"]
    group = case["heads"] // heads
    key = torch.arange(keys, device="cuda")
    seq = torch.arange(n, device="cuda")[:, None]
    there = torch.minimum(key[None], kv_len[:, None] - 1)
    k, v = (_gather(case, s, name, seq, there).transpose(1, 2) for name in ("k", "v"))  # [seq, head, key, dim]
    count = starts[1:] - starts[:-1]
    r = torch.arange(most, device="cuda")
    row = torch.minimum(starts[:-1, None] + r, starts[-1] - 1)
    q = s["q"].float()[row].view(n, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, heads, group * most, dim)
    pos = (kv_len - count)[:, None] + r  # [seq, row]
    seen = key[None, None] < kv_len[:, None, None]
    if case["causal"]:
        seen = seen & (key[None, None] <= pos[..., None])
    if case["window"]:
        seen = seen & (key[None, None] > pos[..., None] - case["window"])
    scores = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(n, heads, group, most, keys)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    scores = scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    o = (scores.view(n, heads, group * most, keys) @ v).view(n, heads, group, most, dim)
    o = torch.where(total > 0, o / total, 0.0)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    use = r[None] < count[:, None]
    out = o.permute(0, 3, 1, 2, 4).reshape(n, most, case["heads"], dim)[use]
    return {"out": out.to(s["q"].dtype), "lse": lse.permute(0, 3, 1, 2).reshape(n, most, case["heads"])[use]}


def _run_sample(case, s):
    n, x = case["n"], s["x"].double()
    rank = torch.arange(n, device="cuda")[None]
    greedy = s["t"] <= 0
    t = torch.where(greedy, torch.ones_like(s["t"]), s["t"]).double()[:, None]
    k = torch.where(greedy, 1, torch.where(s["k"] > 0, s["k"], n))[:, None]
    ordered, at = torch.sort(x, dim=1, descending=True, stable=True)
    w = ((ordered - ordered[:, :1]) / t).exp()
    w = torch.where(rank < k, w, 0.0)
    before = w.cumsum(1) - w
    p = s["p"].double()[:, None]
    kept = (rank < k) & ((p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0)) & (w >= s["m"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, at, torch.where(kept, w, 0.0))
    run = w.cumsum(1)
    ids = (run <= s["u"].double()[:, None] * run[:, -1:]).sum(1, keepdim=True)
    logp = (w.gather(1, ids) / run[:, -1:]).log()
    return {"ids": ids[:, 0].int(), "logp": logp[:, 0].float()}


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "rope":
        return _run_rope(case, state)
    if case["op"] == "write":
        return _run_write(case, state)
    if case["op"] == "read":
        return _run_read(case, state)
    if case["op"] == "attention":
        return _run_attention(case, state)
    return _run_sample(case, state)


# ---- what each pass cannot do without ------------------------------------------------------------------------------------------


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
    if case["op"] == "rope":
        x = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * x * size[case["type"]] + 4 * case["rows"], "flops": 3 * case["rows"] * case["heads"] * case["rot"]}
    if case["op"] == "sample":
        x = case["rows"] * case["n"]
        return {"bytes": x * size[case["type"]] + 28 * case["rows"], "flops": 2 * x}
    new, kv = _lengths(case)
    wide, code = case["kv_heads"] * case["dim"], size[case["cache"]]
    scale = 4 * case["kv_heads"] if case["cache"] in TOP else 0
    if case["op"] in ("write", "read"):
        rows = int(new.sum() if case["op"] == "write" else kv.sum())
        return {"bytes": 2 * rows * (wide * (code + size[case["type"]]) + scale), "flops": 2 * rows * wide}
    rows = int(new.sum())
    pairs = keys = 0
    for m, n in zip(new.tolist(), kv.tolist()):
        pos = np.arange(n - m, n)
        last = pos + 1 if case["causal"] else np.full(m, n)
        first = np.maximum(pos - case["window"] + 1, 0) if case["window"] else np.zeros(m, np.int64)
        pairs += int((last - first).sum())
        keys += int(last.max() - first.min())
    return {"bytes": 2 * keys * (wide * code + scale) + rows * case["heads"] * (2 * case["dim"] * size[case["type"]] + 4),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        spec, half = _rope_spec(case), case["rot"] // 2
        turn = []
        for i in range(half):
            f = math.exp(-2.0 * i / case["rot"] * math.log(10000.0))
            if case["scaling"] == "linear":
                f /= spec["factor"]
            elif case["scaling"] == "bands":
                length = 2 * math.pi / f
                if length > spec["original_len"] / spec["low"]:
                    f /= spec["factor"]
                elif length >= spec["original_len"] / spec["high"]:
                    part = (spec["original_len"] / length - spec["low"]) / (spec["high"] - spec["low"])
                    f = part * f + (1 - part) * f / spec["factor"]
            elif case["scaling"] == "ramp":
                def place(turns):
                    return case["rot"] * math.log(spec["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
                first, last = max(0, math.floor(place(spec["high"]))), min(case["rot"] - 1, math.ceil(place(spec["low"])))
                share = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
                f = share * f / spec["factor"] + (1 - share) * f
            turn.append(f)
        angle = s["pos"].double()[:, None] * torch.tensor(turn, dtype=torch.float64, device="cuda")
        z = torch.polar(torch.full_like(angle, spec.get("magnitude", 1.0)), angle)[:, None]
        x = s["x"].double()
        part = x[..., : case["rot"]]
        if case["inter"]:
            y = torch.view_as_real(torch.view_as_complex(part.reshape(*part.shape[:-1], half, 2).contiguous()) * z).flatten(-2)
        else:
            t = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * z
            y = torch.cat([t.real, t.imag], -1)
        return torch.cat([y, x[..., case["rot"] :]], -1)
    if case["op"] == "sample":
        x, ids, logp = s["x"].double().cpu().numpy(), None, []
        if x.size > 40_000_000:
            return None
        for r in range(case["rows"]):
            t, k, p, m, u = (float(s[c][r]) for c in "tkpmu")
            order = np.argsort(-x[r], kind="stable")
            if t <= 0:
                logp.append(0.0)
                continue
            order = order[: int(k)] if k > 0 else order
            w = np.exp((x[r][order] - x[r][order[0]]) / t)
            if p < 1:
                whole = math.fsum(w) if len(w) < 2000 else w.sum()
                order = order[: int(np.searchsorted(np.cumsum(w), p * whole)) + 1]
                w = w[: len(order)]
            order = np.sort(order[w >= m])
            w = np.exp((x[r][order] - x[r].max()) / t)
            c = np.cumsum(w)
            logp.append(float(np.log(w[np.searchsorted(c, u * c[-1], side="right")] / c[-1])))
        return {"ids": ids, "logp": np.array(logp)}
    starts, kv_len, table = (s[n].cpu().numpy() for n in ("starts", "kv_len", "table"))

    def pages(name, i):
        """A sequence's keys or values in 64 bits, [key, head, dim]."""
        at = torch.from_numpy(table[i][: -(-int(kv_len[i]) // case["page"])].astype(np.int64)).cuda()
        x = s["pool_" + name][at].double()
        x = x.transpose(1, 2) if case["order"] == "head" else x
        if case["cache"] in TOP:
            x = x * s["scale_" + name][at].double().transpose(1, 2)[..., None]
        return x.reshape(-1, case["kv_heads"], case["dim"])[: int(kv_len[i])]

    if case["op"] == "read":
        return {name: torch.cat([pages(name, i) for i in range(case["seqs"])]) for name in ("k", "v")}
    if case["op"] == "write":
        got = {}
        for name in ("k", "v"):
            x = s[name].double()
            pool = torch.zeros(s["pool_" + name].shape, dtype=torch.float64, device="cuda")
            at = np.concatenate([np.arange(kv_len[i] - (starts[i + 1] - starts[i]), kv_len[i]) for i in range(case["seqs"])])
            seq = np.repeat(np.arange(case["seqs"]), starts[1:] - starts[:-1])
            page, slot = (torch.from_numpy(v).cuda() for v in (table[seq, at // case["page"]].astype(np.int64), at % case["page"]))
            if case["cache"] in TOP:
                scale = x.abs().amax(-1) / TOP[case["cache"]]
                kept = torch.zeros(s["scale_" + name].shape, dtype=torch.float64, device="cuda")
                kept[page, :, slot] = scale
                got["scale_" + name] = kept
                x = x / scale[..., None]
                step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0**-6))) - 3)
                x = torch.round(x / step) * step
            if case["order"] == "slot":
                pool[page, slot] = x
            else:
                pool[page, :, slot] = x
            got["pool_" + name] = None if case["cache"] == "i8" else pool
        return got
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    for i in range(case["seqs"]):
        a, b, n = int(starts[i]), int(starts[i + 1]), int(kv_len[i])
        k, v = pages("k", i), pages("v", i)
        back = torch.arange(b - a, 0, -1, device="cuda")[:, None] - (n - torch.arange(n, device="cuda"))[None]  # how far a key lies ahead, negated
        hidden = torch.zeros_like(back, dtype=torch.bool)
        if case["causal"]:
            hidden |= back > 0
        if case["window"]:
            hidden |= back <= -case["window"]
        for h in range(case["kv_heads"]):
            q = s["q"][a:b, h * group : (h + 1) * group].double()
            z = torch.einsum("rgd,nd->rgn", q, k[:, h]) / math.sqrt(case["dim"])
            z = z.masked_fill(hidden[:, None], -math.inf)
            e = torch.logsumexp(z, -1)
            w = torch.exp(z - torch.where(torch.isfinite(e), e, 0.0)[..., None])
            out[a:b, h * group : (h + 1) * group] = torch.einsum("rgn,nd->rgd", w, v[:, h])
            lse[a:b, h * group : (h + 1) * group] = e
    return {"out": out, "lse": lse}
