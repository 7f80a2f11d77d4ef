"""The float operators of a decoder layer that stand beside its fixed-point stages: what is measured of them.

Three operators, each with the direction that training needs:

  rope        rotary positions of queries and keys in one call
  norm        the norms after one branch and before the next, with the branch's gate, residual scale and addition between
  glu         the gated feed-forward block: both projections, the activation and the product

`run` computes them in plain torch operations, or, where `own` is true, through the library's C ABI.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}
GATES = {"none": 0, "channel": 1, "row": 2, "element": 3}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one new token for each of 8 sequences, far into their contexts
        {"name": "rope decode", "op": "rope", "type": "bf16", "batch": 8, "tokens": 1, "q_heads": 32, "k_heads": 32, "head_dim": 128, "rotary_dim": 128,
         "layout": "half", "scaling": "linear", "far": 131072, "backward": False},
        # a prompt of the benchmark layer's length and heads
        {"name": "rope prompt", "op": "rope", "type": "bf16", "batch": 1, "tokens": 2048, "q_heads": 32, "k_heads": 32, "head_dim": 128, "rotary_dim": 128,
         "layout": "half", "scaling": "none", "far": 0, "backward": False},
        # gradients over a ragged batch, half of each head turned, neighbouring pairs, fewer key heads
        {"name": "rope backward part", "op": "rope", "type": "f32", "batch": 3, "tokens": 4097, "q_heads": 40, "k_heads": 8, "head_dim": 128, "rotary_dim": 64,
         "layout": "interleaved", "scaling": "ramp", "far": 32768, "backward": True},
        # the norms of one decoding step
        {"name": "norm decode", "op": "norm", "type": "bf16", "gains": "bf16", "rows": 8, "cols": 4096, "post": True, "gate": "channel", "backward": False},
        # between the attention and the feed-forward block of the benchmark layer
        {"name": "norm prompt", "op": "norm", "type": "bf16", "gains": "bf16", "rows": 2048, "cols": 4096, "post": True, "gate": "channel", "backward": False},
        # its gradients on a long batch of the wider model, gains in 32 bits
        {"name": "norm backward", "op": "norm", "type": "bf16", "gains": "f32", "rows": 8192, "cols": 5120, "post": True, "gate": "channel", "backward": True},
        # gradients with a gate for each value, rows of an odd length
        {"name": "norm backward odd", "op": "norm", "type": "f32", "gains": "f32", "rows": 1023, "cols": 4099, "post": True, "gate": "element", "backward": True},
        # one token through the benchmark layer's feed-forward block: latency of the two weights' read
        {"name": "glu decode", "op": "glu", "type": "bf16", "tokens": 1, "in": 4096, "hidden": 11008, "act": "silu", "keep": False, "backward": False},
        # a batch of sequences that each decode one token, the wider model
        {"name": "glu decode batch", "op": "glu", "type": "f16", "tokens": 48, "in": 5120, "hidden": 13824, "act": "gelu_tanh", "keep": False, "backward": False},
        # the benchmark layer's prompt, both projections kept for the gradients
        {"name": "glu prompt", "op": "glu", "type": "bf16", "tokens": 2048, "in": 4096, "hidden": 11008, "act": "silu", "keep": True, "backward": False},
        # its gradients
        {"name": "glu backward", "op": "glu", "type": "bf16", "tokens": 2048, "in": 4096, "hidden": 11008, "act": "silu", "keep": True, "backward": True},
        # gradients at sizes that fill no tile and whose rows start at odd addresses
        {"name": "glu backward odd", "op": "glu", "type": "f16", "tokens": 777, "in": 1001, "hidden": 2731, "act": "gelu", "keep": True, "backward": True},
    ]


def _spread(rng, low, high, step=1):
    """a whole multiple of step, its logarithm spread evenly over the range"""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 0.99)))
    return max(low, min(high, int(v / step + 0.5) * step or step))


def draw(rng):
    kind = rng.choice(["rope", "norm", "glu", "glu"])
    backward = rng.random() < 0.5
    if kind == "rope":
        head_dim = rng.choice([64, 80, 96, 128, 192, 256])
        case = {"op": "rope", "type": rng.choice(list(DTYPES)), "batch": rng.randint(1, 8), "tokens": _spread(rng, 1, 4096), "q_heads": rng.randint(1, 40),
                "k_heads": rng.choice([1, 2, 4, 8, 32]), "head_dim": head_dim, "rotary_dim": rng.choice([head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)]),
                "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "ntk", "ramp"]),
                "far": rng.choice([0, 4096, 131072]), "backward": backward}
        most = 8192 * 5120 // ((case["q_heads"] + case["k_heads"]) * head_dim)   # no more values than the largest listed call
        case["tokens"] = max(1, min(case["tokens"], most // case["batch"]))
        return case
    if kind == "norm":
        cols = _spread(rng, 64, 13824, rng.choice([1, 8, 64]))
        return {"op": "norm", "type": rng.choice(list(DTYPES)), "gains": rng.choice(["f32", "same"]), "rows": min(_spread(rng, 1, 8192), 8192 * 2560 // cols),
                "cols": cols, "post": rng.random() < 0.7, "gate": rng.choice(list(GATES)), "backward": backward}
    width = _spread(rng, 64, 5120, rng.choice([1, 8, 128]))
    hidden = _spread(rng, 64, 13824, rng.choice([1, 8, 128]))
    tokens = min(_spread(rng, 1, 4096), 2048 * 4096 * 11008 // (width * hidden))
    return {"op": "glu", "type": rng.choice(["f16", "bf16"]), "tokens": tokens, "in": width, "hidden": hidden, "act": rng.choice(list(ACTIVATIONS)),
            "keep": True if backward else rng.random() < 0.5, "backward": backward}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------


def _frequencies(case):
    """radians a position of each pair (64 bits, on the host) and the factor on the turned values"""
    n = case["rotary_dim"]
    base, factor, original = 10000.0, 4.0, 4096.0
    if case["scaling"] == "ntk" and n > 2:
        base *= factor ** (n / (n - 2))
    f = [base ** (-2.0 * i / n) for i in range(n // 2)]
    if case["scaling"] == "linear":
        f = [v / factor for v in f]
    if case["scaling"] == "ramp":   # pairs that turn often over the original context stay, slow ones are stretched, a ramp between
        at = lambda turns: n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0.0), min(math.ceil(at(1.0)), n - 1.0)
        share = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(n // 2)]
        f = [v / factor * s + v * (1 - s) for v, s in zip(f, share)]
    return f, (0.1 * math.log(factor) + 1.0 if case["scaling"] == "ramp" else 1.0)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = DTYPES[case["type"]]
    rand = lambda *shape, by=1.0, dtype=t: (torch.randn(*shape, generator=g, device="cuda") * by).to(dtype)  # noqa: E731
    empty = lambda *shape, dtype=t: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731
    s = {"case": case}
    if case["op"] == "rope":
        b, n, d = case["batch"], case["tokens"], case["head_dim"]
        f, s["magnitude"] = _frequencies(case)
        s["inv_freq"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        s["q"], s["k"] = rand(b, n, case["q_heads"], d), rand(b, n, case["k_heads"], d)
        first = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device="cuda")   # every sequence has its own past
        s["positions"] = first + torch.arange(n, device="cuda")
        s["q_out"], s["k_out"] = empty(*s["q"].shape), empty(*s["k"].shape)
        return s
    if case["op"] == "norm":
        rows, cols, kind = case["rows"], case["cols"], case["gate"]
        w = t if case["gains"] == "same" else DTYPES[case["gains"]]
        s["wide"] = 1.0 + 9.0 * (torch.rand(cols, generator=g, device="cuda") < 0.01)   # a few channels stand out, as in trained models
        s["y"] = (rand(rows, cols, dtype=torch.float32) * s["wide"]).to(t)
        s["post_gain"] = (1 + rand(cols, by=0.1, dtype=torch.float32)).to(w) if case["post"] else None
        s["pre_gain"] = (1 + rand(cols, by=0.1, dtype=torch.float32)).to(w)
        shape, wt = {"none": (None, t), "channel": ((cols,), w), "row": ((rows,), t), "element": ((rows, cols), t)}[kind]
        s["gate"] = None if shape is None else rand(*shape, by=0.5, dtype=wt)
        s["scale"], s["eps"] = 0.7, 1e-5
        x = (rand(rows, cols, dtype=torch.float32) * s.pop("wide")).to(t)
        if case["backward"]:
            s["r"], s["dz"], s["dr"] = x, rand(rows, cols), rand(rows, cols)
            s["dx"], s["dy"], s["dpre"] = empty(rows, cols), empty(rows, cols), empty(cols, dtype=w)
            s["dpost"] = empty(cols, dtype=w) if case["post"] else None
            s["dgate"] = None if shape is None else empty(*shape, dtype=wt)
        else:
            s["x"], s["r"], s["z"], s["inv"] = x, empty(rows, cols), empty(rows, cols), empty(rows, dtype=torch.float32)
        return s
    n, e, f = case["tokens"], case["in"], case["hidden"]
    s["x"] = rand(n, e)
    s["w_gate"], s["w_up"] = rand(e, f, by=e ** -0.5), rand(e, f, by=e ** -0.5)
    if case["backward"]:
        s["gate"], s["up"], s["dh"] = rand(n, f), rand(n, f), rand(n, f)
        s["dx"], s["dw_gate"], s["dw_up"] = empty(n, e), empty(e, f), empty(e, f)
    else:
        s["h"] = empty(n, f)
        s["gate"], s["up"] = (empty(n, f), empty(n, f)) if case["keep"] else (None, None)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------------------------


def _turn(x, cos, sin, case):
    n, t = case["rotary_dim"], x.dtype
    x = x.float()
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if case["layout"] == "interleaved" else (x[..., :n // 2], x[..., n // 2:n])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((c, d), -1).flatten(-2) if case["layout"] == "interleaved" else torch.cat((c, d), -1)
    return torch.cat((turned, x[..., n:]), -1).to(t)


def _plain_rope(s):
    angle = (s["positions"].double()[..., None] * s["inv_freq"])[:, :, None, :]   # far positions: 32 bits lose the angle
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    sin = -sin if s["case"]["backward"] else sin
    return [_turn(s["q"], cos, sin, s["case"]), _turn(s["k"], cos, sin, s["case"])]


def _wide(s, *names):
    return [None if s[n] is None else s[n].float() for n in names]


def _plain_norm(s):
    kind, t = s["case"]["gate"], s["y"].dtype
    y, post, pre, gate = _wide(s, "y", "post_gain", "pre_gain", "gate")
    gate = 1.0 if gate is None else gate[:, None] if kind == "row" else gate
    post_inv = torch.rsqrt((y * y).mean(1, keepdim=True) + s["eps"])
    n = y if post is None else y * post_inv * post
    if not s["case"]["backward"]:
        r = s["x"].float() + s["scale"] * gate * n
        inv = torch.rsqrt((r * r).mean(1, keepdim=True) + s["eps"])
        return [r.to(t), (r * inv * pre).to(t), inv[:, 0]]
    r, dz, dr = _wide(s, "r", "dz", "dr")
    inv = torch.rsqrt((r * r).mean(1, keepdim=True) + s["eps"])
    p = dz * pre
    d = dr + inv * (p - r * (inv * inv * (p * r).mean(1, keepdim=True)))
    dn = s["scale"] * gate * d
    dy = dn
    if post is not None:
        p = dn * post
        dy = post_inv * (p - y * (post_inv * post_inv * (p * y).mean(1, keepdim=True)))
    out = [d.to(t), dy.to(t), (dz * r * inv).sum(0).to(s["pre_gain"].dtype)]
    if post is not None:
        out.append((dn * y * post_inv).sum(0).to(s["post_gain"].dtype))
    if kind != "none":
        dg = s["scale"] * d * n
        dg = dg.sum(0) if kind == "channel" else dg.sum(1) if kind == "row" else dg
        out.append(dg.to(s["gate"].dtype))
    return out


def _activation(g, kind):
    """act(g) and its derivative"""
    if kind == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    if kind == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        th = torch.tanh(k * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * k * (1 + 3 * 0.044715 * g * g)
    return torch.where(g > 0, g, 0.0), (g > 0).to(g.dtype)


def _plain_glu(s):
    t = s["x"].dtype
    x, wg, wu = _wide(s, "x", "w_gate", "w_up")
    if not s["case"]["backward"]:
        g, u = x @ wg, x @ wu
        h = (_activation(g, s["case"]["act"])[0] * u).to(t)
        return [h, g.to(t), u.to(t)] if s["case"]["keep"] else [h]
    g, u, dh = _wide(s, "gate", "up", "dh")
    a, da = _activation(g, s["case"]["act"])
    dg, du = dh * u * da, dh * a
    return [(dg @ wg.T + du @ wu.T).to(t), (x.T @ dg).to(t), (x.T @ du).to(t)]


# ---- the library's calls -------------------------------------------------------------------------------------------------------------------


def _at(x):
    return None if x is None else x.data_ptr()


def _own_rope(s):
    z, c = importlib.import_module("zkllm-ccs2024_b200"), s["case"]
    q, k, pos = s["q"], s["k"], s["positions"]
    both = z.rope_tensors(*((x.data_ptr(), y.data_ptr(), x.shape[2], x.stride()[:3], y.stride()[:3]) for x, y in ((q, s["q_out"]), (k, s["k_out"]))))
    z.call("zkb_rope", CODES[c["type"]], both, 2, c["batch"], c["tokens"], c["head_dim"], c["rotary_dim"], int(c["layout"] == "interleaved"),
           s["inv_freq"].data_ptr(), s["magnitude"], pos.data_ptr(), pos.stride(0), 0, int(c["backward"]), torch.cuda.current_stream().cuda_stream)
    return [s["q_out"], s["k_out"]]


def _own_norm(s):
    z, c = importlib.import_module("zkllm-ccs2024_b200"), s["case"]
    cols, kind = c["cols"], GATES[c["gate"]]
    t = CODES[c["type"]]
    w = t if c["gains"] == "same" else CODES[c["gains"]]
    stream = torch.cuda.current_stream().cuda_stream
    if not c["backward"]:
        z.call("zkb_block_norm", t, w, c["rows"], cols, _at(s["x"]), cols, _at(s["y"]), cols, int(c["post"]), _at(s["post_gain"]), kind, _at(s["gate"]), cols,
               s["scale"], 1, _at(s["pre_gain"]), s["eps"], _at(s["r"]), cols, _at(s["z"]), cols, None, _at(s["inv"]), stream)
        return [s["r"], s["z"], s["inv"]]
    z.call("zkb_block_norm_backward", t, w, c["rows"], cols, _at(s["r"]), cols, _at(s["y"]), cols, int(c["post"]), _at(s["post_gain"]), kind, _at(s["gate"]),
           cols, s["scale"], 1, _at(s["pre_gain"]), s["eps"], _at(s["dz"]), cols, _at(s["dr"]), cols, _at(s["dx"]), cols, _at(s["dy"]), cols,
           _at(s["dgate"]), cols, _at(s["dpost"]), _at(s["dpre"]), stream)
    return [x for x in (s["dx"], s["dy"], s["dpre"], s["dpost"], s["dgate"]) if x is not None]


def _own_glu(s):
    z, c = importlib.import_module("zkllm-ccs2024_b200"), s["case"]
    n, e, f = c["tokens"], c["in"], c["hidden"]
    t, act = CODES[c["type"]], ACTIVATIONS[c["act"]]
    stream = torch.cuda.current_stream().cuda_stream
    if not c["backward"]:
        z.call("zkb_glu", t, act, n, e, f, _at(s["x"]), e, _at(s["w_gate"]), f, _at(s["w_up"]), f, _at(s["h"]), f, _at(s["gate"]), f, _at(s["up"]), f, stream)
        return [s["h"], s["gate"], s["up"]] if c["keep"] else [s["h"]]
    z.call("zkb_glu_backward", t, act, n, e, f, _at(s["x"]), e, _at(s["w_gate"]), f, _at(s["w_up"]), f, _at(s["gate"]), f, _at(s["up"]), f, _at(s["dh"]), f,
           _at(s["dx"]), e, _at(s["dw_gate"]), f, _at(s["dw_up"]), f, stream)
    return [s["dx"], s["dw_gate"], s["dw_up"]]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "norm": _own_norm, "glu": _own_glu}[op](state)
    return {"rope": _plain_rope, "norm": _plain_norm, "glu": _plain_glu}[op](state)


# ---- floors and the definition in 64 bits ---------------------------------------------------------------------------------------------------


def work(case):
    b = BYTES[case["type"]]
    if case["op"] == "rope":
        rows = case["batch"] * case["tokens"] * (case["q_heads"] + case["k_heads"])
        return {"bytes": 2 * b * rows * case["head_dim"] + 8 * case["batch"] * case["tokens"] + 4 * case["rotary_dim"], "flops": 3 * rows * case["rotary_dim"]}
    if case["op"] == "norm":
        rows, cols, wb = case["rows"], case["cols"], b if case["gains"] == "same" else BYTES[case["gains"]]
        vectors = (1 + case["post"]) * cols * wb
        gate = {"none": 0, "channel": cols * wb, "row": rows * b, "element": rows * cols * b}[case["gate"]]
        if not case["backward"]:
            return {"bytes": 4 * b * rows * cols + vectors + gate + 4 * rows, "flops": 10 * rows * cols}
        return {"bytes": 6 * b * rows * cols + 2 * (vectors + gate), "flops": 26 * rows * cols}
    n, e, f = case["tokens"], case["in"], case["hidden"]
    if not case["backward"]:
        return {"bytes": b * (n * e + 2 * e * f + (3 if case["keep"] else 1) * n * f), "flops": 4 * n * e * f}
    return {"bytes": b * (2 * n * e + 4 * e * f + 3 * n * f), "flops": 8 * n * e * f}


def _exact_rope(s):
    c = s["case"]
    half = c["rotary_dim"] // 2
    angle = (s["positions"].double().unsqueeze(-1) * s["inv_freq"]).unsqueeze(2) * (-1.0 if c["backward"] else 1.0)
    unit = torch.polar(torch.full_like(angle, s["magnitude"]), angle)
    out = []
    for x in (s["q"].double(), s["k"].double()):
        pairs = x[..., :2 * half].unflatten(-1, (half, 2) if c["layout"] == "interleaved" else (2, half))
        dim = -1 if c["layout"] == "interleaved" else -2
        turned = torch.complex(pairs.select(dim, 0), pairs.select(dim, 1)) * unit
        x[..., :2 * half] = torch.stack((turned.real, turned.imag), dim).flatten(-2)
        out.append(x)
    return out


def _exact_norm(s):
    """the gradients come from torch's own differentiation of the forward formula"""
    c = s["case"]
    y, post, pre, gate = [None if s[n] is None else s[n].double().requires_grad_(c["backward"]) for n in ("y", "post_gain", "pre_gain", "gate")]
    norm = lambda v, w: v / (v.pow(2).mean(-1, keepdim=True) + s["eps"]).sqrt() * w  # noqa: E731
    branch = y if post is None else norm(y, post)
    if gate is not None:
        branch = branch * (gate.unsqueeze(1) if c["gate"] == "row" else gate)
    branch = branch * s["scale"]
    if not c["backward"]:
        r = s["x"].double() + branch
        return [r, norm(r, pre), 1 / (r.pow(2).mean(-1) + s["eps"]).sqrt()]
    r = s["r"].double()
    x = (r - branch.detach()).requires_grad_(True)   # the stream before the branch, so that the sum is the given r
    total = x + branch
    leaves = [v for v in (x, y, pre, post, gate) if v is not None]
    return list(torch.autograd.grad([total, norm(total, pre)], leaves, [s["dr"].double(), s["dz"].double()]))


def _exact_glu(s):
    c = s["case"]
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
           "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[c["act"]]
    x, wg, wu = (s[n].double() for n in ("x", "w_gate", "w_up"))
    if not c["backward"]:
        g, u = torch.mm(x, wg), torch.mm(x, wu)
        return [act(g) * u, g, u] if c["keep"] else [act(g) * u]
    g, u = (s[n].double().requires_grad_(True) for n in ("gate", "up"))
    dg, du = torch.autograd.grad(act(g) * u, (g, u), s["dh"].double())
    return [torch.mm(dg, wg.t()) + torch.mm(du, wu.t()), torch.mm(x.t(), dg), torch.mm(x.t(), du)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "norm": _exact_norm, "glu": _exact_glu}[case["op"]](s)
