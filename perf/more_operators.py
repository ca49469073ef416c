"""Cases of the operators between the serving calls: residual addition with a root-mean-square norm (to 16 bits or to 8-bit floats with a scale
a row), the product of rows with a weight matrix with bias, activation and residual, and the gated pair of products of a feed-forward block.

``run`` computes them in plain torch operations, or, with ``own`` set, through the framework's device-pointer calls.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
CODES = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 4}  # of the framework's calls
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
ACTS = {"none": -1, "gelu": 2, "silu": 3, "relu": 4, "tanh": 5, "sigmoid": 6}
EPS = 1e-5


def listed():
    return [
        # before a layer's projections, one new token of each of 32 conversations
        dict(name="norm step", op="norm", rows=32, n=4096, type="bf16", to="bf16", residual=True, norm=True),
        # the same for a batch of prompts whose next product runs in 8 bits
        dict(name="norm prompt", op="norm", rows=8192, n=4096, type="bf16", to="e4m3", residual=True, norm=True),
        # the hidden rows of a feed-forward block, ragged, made 8 bits wide for the product that follows
        dict(name="codes prompt", op="norm", rows=5003, n=12288, type="f16", to="e4m3", residual=False, norm=False),
        # queries, keys and values of one token of one conversation with the framework's decoder
        dict(name="linear one token", op="linear", rows=1, n_in=768, n_out=2304, type="f16", to="f16", bias=True, act="none", residual=False),
        # the projection behind the attention of a batch of conversations, added to what passes by
        dict(name="linear step", op="linear", rows=48, n_in=4096, n_out=4096, type="bf16", to="bf16", bias=False, act="none", residual=True),
        # the logits of the next tokens, vocabulary of the framework's decoder, in fp32 for the sampling
        dict(name="linear logits", op="linear", rows=16, n_in=4096, n_out=32000, type="bf16", to="f32", bias=False, act="none", residual=False),
        # the wide half of a feed-forward block without a gate over a batch of prompts
        dict(name="linear prompt", op="linear", rows=8192, n_in=4096, n_out=16384, type="bf16", to="bf16", bias=True, act="gelu", residual=False),
        # the way back from a wide feed-forward block in 8 bits, ragged prompts
        dict(name="linear prompt 8 bits", op="linear", rows=5003, n_in=12288, n_out=4096, type="e4m3", to="bf16", bias=False, act="none", residual=True),
        # a feed-forward block for the next tokens of a few conversations
        dict(name="gated step", op="gated", rows=8, n_in=4096, n_out=12288, type="bf16", to="bf16", bias=False, act="silu"),
        # the same in 8 bits for a large batch of conversations
        dict(name="gated step 8 bits", op="gated", rows=128, n_in=4096, n_out=12288, type="e4m3", to="bf16", bias=False, act="silu"),
        # ... for ragged prompts
        dict(name="gated prompt", op="gated", rows=3001, n_in=4096, n_out=12288, type="bf16", to="bf16", bias=False, act="silu"),
        # ... in 8 bits, odd sizes, with biases
        dict(name="gated prompt 8 bits", op="gated", rows=6000, n_in=5120, n_out=13001, type="e4m3", to="f16", bias=True, act="gelu"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "gated", "gated"])
    if op == "norm":
        n = _log(rng, 33, 16384)
        n = n if rng.random() < 0.4 else -(-n // 64) * 64
        case = dict(op=op, rows=_log(rng, 1, min(16384, 60_000_000 // n)), n=n, type=rng.choice(["f32", "f16", "bf16", "bf16"]))
        case["to"] = rng.choice([case["type"], "bf16", "f16", "e4m3", "e4m3"])
        case["norm"] = case["to"] != "e4m3" or rng.random() < 0.7
        case["residual"] = case["norm"] and rng.random() < 0.7
        return case
    n_in, n_out = _log(rng, 64, 16384), _log(rng, 64, 32000 if op == "linear" else 16384)
    if rng.random() < 0.7:
        n_in, n_out = -(-n_in // 64) * 64, -(-n_out // 64) * 64
    most = min(1_000_000_000_000 // (2 * n_in * n_out * (2 if op == "gated" else 1)), 134_000_000 // n_out)
    kind = rng.choice(["f16", "bf16", "bf16", "e4m3", "e4m3"])
    case = dict(op=op, rows=_log(rng, 1, max(1, min(most, 16384))), n_in=n_in, n_out=n_out, type=kind, to=rng.choice(["f32", "f16", "bf16", "bf16"]),
                bias=rng.random() < 0.4, act=rng.choice(["silu", "gelu"] if op == "gated" else ["none", "none", "gelu", "relu", "tanh"]))
    if op == "linear":
        case["residual"] = rng.random() < 0.4
    return case


def _wide(n):
    """The elements from one row of an operand to the next: rows start on 16 bytes in every type."""
    return -(-n // 16) * 16


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    rows, to = case["rows"], TYPES[case["to"]]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def operand(count, wide, scale):
        """Rows of an operand, and the scale of each where it is held in 8 bits."""
        if case["type"] != "e4m3":
            x = torch.zeros(count, _wide(wide), dtype=TYPES[case["type"]], device="cuda")
            x[:, :wide] = normal(count, wide, scale=scale)
            return x[:, :wide], None
        x = torch.zeros(count, _wide(wide), device="cuda")
        x[:, :wide] = normal(count, wide, scale=112.0).clamp_(-448.0, 448.0)
        return x.to(TYPES["e4m3"])[:, :wide], (0.5 + torch.rand(count, generator=g, device="cuda")) * (scale / 112.0)

    if case["op"] == "norm":
        n, kind = case["n"], TYPES[case["type"]]
        s["x"] = normal(rows, n, scale=2.0, dtype=kind)
        if case["residual"]:
            s["residual"] = normal(rows, n, dtype=kind)
            s["sum"] = torch.empty_like(s["x"])
        if case["norm"]:
            s["gamma"] = 1.0 + normal(n, scale=0.1)
        s["y"] = torch.empty(rows, _wide(n), dtype=to, device="cuda")[:, :n]
        if case["to"] == "e4m3":
            s["scale"] = torch.empty(rows, device="cuda")
    else:
        n_in, n_out = case["n_in"], case["n_out"]
        s["x"], s["x_scale"] = operand(rows, n_in, 1.0)
        for name in ("w", "up") if case["op"] == "gated" else ("w",):
            s[name], s[name + "_scale"] = operand(n_out, n_in, 1.0 / math.sqrt(n_in))
            s[name + "_bias"] = normal(n_out, scale=0.1) if case["bias"] else None
        if case.get("residual"):
            s["residual"] = normal(rows, n_out, dtype=to)
        s["y"] = torch.empty(rows, n_out, dtype=to, device="cuda")
    if own:
        s["own"] = _own_plan(case, s)
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------------


def _own_plan(case, s):
    """What a program keeps: the description of its buffers."""
    from mimir_framework_b200 import runtime as rt

    rt.init(0)

    def at(name):
        return s[name].data_ptr() if s.get(name) is not None else None

    def step(name):
        return s[name].stride(0) if s.get(name) is not None else 0

    if case["op"] == "norm":
        return rt.norm_rows(x=at("x"), y=at("y"), rows=case["rows"], n=case["n"], type=CODES[case["type"]], y_type=CODES[case["to"]], x_stride=step("x"),
                            y_stride=step("y"), gamma=at("gamma"), residual=at("residual"), residual_stride=step("residual"), sum=at("sum"),
                            sum_stride=step("sum"), y_scale=at("scale"), norm=case["norm"], eps=EPS)
    return rt.linear(x=at("x"), w=at("w"), out=at("y"), rows=case["rows"], n_in=case["n_in"], n_out=case["n_out"], type=CODES[case["type"]],
                     out_type=CODES[case["to"]], x_stride=step("x"), w_stride=step("w"), out_stride=step("y"), x_scale=at("x_scale"),
                     w_scale=at("w_scale"), bias=at("w_bias"), up=at("up"), up_stride=step("up"), up_scale=at("up_scale"), up_bias=at("up_bias"),
                     residual=at("residual"), residual_stride=step("residual"), activation=ACTS[case["act"]])


def _run_own(case, s):
    from mimir_framework_b200 import runtime as rt

    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "norm":
        rt.dev_norm_rows(s["own"], stream)
    elif case["op"] == "linear":
        rt.dev_linear(s["own"], stream)
    else:
        rt.dev_gated_linear(s["own"], stream)
    return {name: s[name] for name in ("sum", "y", "scale") if name in s}


# ---- the plain forms --------------------------------------------------------------------------------------------------------


def _run_norm(case, s):
    x, got = s["x"].float(), {}
    if case["residual"]:
        x = x + s["residual"].float()
        got["sum"] = x.to(s["x"].dtype)
    if case["norm"]:
        x = x * (1.0 / ((x * x).sum(-1, keepdim=True) / case["n"] + EPS).sqrt()) * s["gamma"]
    if case["to"] == "e4m3":
        scale = x.abs().amax(-1) * (1.0 / 448.0)
        x = torch.where(scale[:, None] > 0, x / scale[:, None], 0.0)
        got["scale"] = scale
    got["y"] = x.to(TYPES[case["to"]])
    return {name: got[name] for name in ("sum", "y", "scale") if name in got}


def _act(x, act):
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "relu":
        return x.clamp_min(0.0)
    return torch.tanh(x) if act == "tanh" else x


def _product(s, name):
    y = s["x"].float() @ s[name].float().t()
    if s[name + "_scale"] is not None:
        y = y * s["x_scale"][:, None] * s[name + "_scale"]
    return y if s[name + "_bias"] is None else y + s[name + "_bias"]


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "norm":
        return _run_norm(case, state)
    y = _act(_product(state, "w"), case["act"])
    if case["op"] == "gated":
        y = y * _product(state, "up")
    elif case["residual"]:
        y = y + state["residual"].float()
    return {"y": y.to(TYPES[case["to"]])}


# ---- what each pass cannot do without ------------------------------------------------------------------------------------------


def work(case):
    rows = case["rows"]
    if case["op"] == "norm":
        each = SIZE[case["type"]] * (3 if case["residual"] else 1) + SIZE[case["to"]]
        return {"bytes": rows * case["n"] * each + (4 * case["n"] if case["norm"] else 0) + (4 * rows if case["to"] == "e4m3" else 0),
                "flops": rows * case["n"] * (6 if case["norm"] else 2)}
    pair = 2 if case["op"] == "gated" else 1
    n_in, n_out = case["n_in"], case["n_out"]
    size = (rows + pair * n_out) * (n_in * SIZE[case["type"]] + (4 if case["type"] == "e4m3" else 0))
    size += rows * n_out * SIZE[case["to"]] * (2 if case.get("residual") else 1) + (4 * pair * n_out if case["bias"] else 0)
    return {"bytes": size, "flops": 2 * rows * n_in * n_out * pair}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        got, v = {}, s["x"].to(torch.float64)
        if case["residual"]:
            v = torch.add(v, s["residual"].to(torch.float64))
            got["sum"] = v
        if case["norm"]:
            length = torch.linalg.vector_norm(v, dim=1)
            v = torch.einsum("rn,r,n->rn", v, torch.rsqrt(length**2 / case["n"] + EPS), s["gamma"].to(torch.float64))
        if case["to"] == "e4m3":
            scale = torch.linalg.vector_norm(v, ord=math.inf, dim=1) / 448.0
            v = v / torch.where(scale > 0, scale, 1.0)[:, None]
            place = torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3.0  # of the last of the four bits
            return {name: x for name, x in (("sum", got.get("sum")), ("y", torch.ldexp(torch.round(torch.ldexp(v, -place)), place)), ("scale", scale))
                    if name != "sum" or "sum" in got}
        return got | {"y": v}

    def projected(name):
        w, x = s[name].to(torch.float64), s["x"].to(torch.float64)
        if s[name + "_scale"] is not None:
            w, x = w.mul_(s[name + "_scale"].to(torch.float64)[:, None]), x.mul_(s["x_scale"].to(torch.float64)[:, None])
        bias = s[name + "_bias"]
        return torch.matmul(x, w.T) if bias is None else torch.addmm(bias.to(torch.float64), x, w.T)

    z = projected("w")
    if case["act"] == "gelu":
        z = z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * z * (1.0 + 0.044715 * z**2))
    elif case["act"] == "silu":
        z = z * torch.sigmoid(z)
    elif case["act"] == "relu":
        z = torch.where(z > 0, z, 0.0)
    elif case["act"] == "tanh":
        z = 1.0 - 2.0 / (torch.exp(2.0 * z) + 1.0)
    if case["op"] == "gated":
        z = z * projected("up")
    return {"y": z + s["residual"].to(torch.float64) if case["residual"] else z} if case["op"] == "linear" else {"y": z}
