"""GPU: the float operators of a layer against their formulas in 64 bits.

Tolerances.  A result that is rounded once to a type is off by at most half a step, h = eps / 2 relative to its value.  What the
32-bit arithmetic before it adds is bounded term by term: a sum of n products of 32-bit values, in whatever order, is off by at most
about (n + 2) 2^-24 times the sum of the terms' magnitudes; with random signs and the trees used here it is far less, so the bounds
below take sqrt(n) + 8 for n, which a lost term or a wrong index exceeds by orders of magnitude."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32 = 2.0 ** -24
TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
GATES = ("none", "channel", "row", "element")
ACTS = ("silu", "gelu", "gelu_tanh", "relu")


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """half a step among the type's smallest values"""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def near(got, want, t, slack):
    """|got - want| <= half a step of want + slack (slack: the bound on what the 32-bit arithmetic adds, by value)"""
    want, slack = want.double(), torch.as_tensor(slack, dtype=torch.float64, device=want.device)
    off = (got.double() - want).abs()
    lim = half_step(t) * (want.abs() + slack) + slack + tiny(t)
    worst = (off - lim).max().item() if off.numel() else 0.0
    assert worst <= 0.0, f"off by {off.max().item():.3g}, {worst:.3g} over the bound"


def stream():
    return torch.cuda.current_stream().cuda_stream


def at(x):
    return None if x is None else x.data_ptr()


# ---- rotary positions -------------------------------------------------------------------------------------------------------------


def rope_want(x, pos, freq, mag, rotary, interleaved, backward):
    """x [b, t, h, d] in 64 bits"""
    x = x.double().clone()
    ang = (pos.double()[..., None] * freq)[:, :, None, :] * (-1 if backward else 1)
    c, s = ang.cos() * mag, ang.sin() * mag
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])
    y = x.clone()
    if interleaved:
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = a * c - b * s, b * c + a * s
    size = x.abs()
    both = a.abs() + b.abs()
    if interleaved:
        size[..., 0:rotary:2] = size[..., 1:rotary:2] = both
    else:
        size[..., :rotary // 2] = size[..., rotary // 2:rotary] = both
    size[..., rotary:] = 0          # copied values are the same
    return y, size * mag


def rope_call(z, code, tensors, b, n, d, rotary, interleaved, freq, mag, pos, stride, first, backward, st=None):
    arr = z.rope_tensors(*((x.data_ptr(), y.data_ptr(), x.shape[2], x.stride()[:3], y.stride()[:3]) for x, y in tensors))
    z.call("zkb_rope", code, arr, len(tensors), b, n, d, rotary, int(interleaved), freq.data_ptr(), mag, at(pos), stride, first, int(backward),
           stream() if st is None else st)


def rope_freq(rotary, base=10000.0):
    return torch.tensor([base ** (-2.0 * i / rotary) for i in range(rotary // 2)], dtype=torch.float64, device="cuda")


# the angle is exact to 2^-24 of a turn or better, sine and cosine to 2 steps of 32 bits, two products and a sum: 16 steps of 32 bits
ROPE_SLACK = 16 * F32


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("b,n,hq,hk,d,rotary", [(1, 1, 1, 1, 2, 2), (2, 1, 32, 8, 128, 128), (3, 33, 5, 1, 96, 64), (1, 257, 4, 4, 80, 30), (2, 7, 3, 2, 61, 22),
                                                (1, 2, 1, 1, 4096, 4096), (1, 5, 2, 1, 6, 2), (4, 600, 2, 2, 64, 64)])
def test_rope(zkb, kind, interleaved, b, n, hq, hk, d, rotary):
    code, t = TYPES[kind]
    g = gen(b * 1000 + n + d)
    freq = rope_freq(rotary)
    pos = torch.randint(-5, 200000, (b, n), generator=g, device="cuda")
    for backward in (False, True):
        q, k = (torch.randn(b, n, h, d, generator=g, device="cuda").to(t) for h in (hq, hk))
        qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
        rope_call(zkb, code, [(q, qo), (k, ko)], b, n, d, rotary, interleaved, freq, 1.25, pos, n, 0, backward)
        for x, y in ((q, qo), (k, ko)):
            want, size = rope_want(x, pos, freq, 1.25, rotary, interleaved, backward)
            near(y, want, t, ROPE_SLACK * size)
            assert torch.equal(y[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("kind", ("f32", "bf16"))
@pytest.mark.parametrize("shift", (0, 1, 4))
def test_rope_strides_in_place_and_shared_positions(zkb, kind, shift):
    """[batch, head, token, dim] views of wider buffers, at addresses off by `shift` elements, in place; positions shared by the batch, or
    counted from a start; what lies around the tensors stays as it was"""
    code, t = TYPES[kind]
    b, n, h, d, rotary = 2, 19, 3, 64, 48
    freq, g = rope_freq(rotary), gen(3)
    buf = torch.randn(b * h * n * (d + 8) + 16, generator=g, device="cuda").to(t)
    view = buf[shift:shift + b * h * n * (d + 8)].view(b, h, n, d + 8)[..., :d].transpose(1, 2)
    before = buf.clone()
    old = before[shift:shift + b * h * n * (d + 8)].view(b, h, n, d + 8)[..., :d].transpose(1, 2)
    pos = torch.arange(n, device="cuda") * 3 + 100
    rope_call(zkb, code, [(view, view)], b, n, d, rotary, False, freq, 1.0, pos, 0, 0, False)
    want, size = rope_want(old, pos.expand(b, n), freq, 1.0, rotary, False, False)
    near(view, want, t, ROPE_SLACK * size)
    touched = torch.zeros_like(buf, dtype=torch.bool)
    touched[shift:shift + b * h * n * (d + 8)].view(b, h, n, d + 8)[..., :d] = True
    assert torch.equal(buf[~touched], before[~touched])
    out = torch.empty(b, n, h, d, device="cuda", dtype=t)
    rope_call(zkb, code, [(old, out)], b, n, d, rotary, True, freq, 1.0, None, 0, 1 << 40, True)
    want, size = rope_want(old, ((1 << 40) + torch.arange(n, device="cuda")).expand(b, n), freq, 1.0, rotary, True, True)
    # at position 2^40 the 64-bit product of the reference itself is off by 2^40 2^-53 radians, and so is the kernel's
    near(out, want, t, (ROPE_SLACK + 2.0 ** -12) * size)


def test_rope_backward_turns_back(zkb):
    """the gradient's turn undoes the forward one, and <R x, y> = <x, R^T y>"""
    b, n, h, d = 2, 40, 3, 32
    g, freq = gen(5), rope_freq(d)
    pos = torch.randint(0, 100000, (b, n), generator=g, device="cuda")
    x, y = (torch.randn(b, n, h, d, generator=g, device="cuda") for _ in range(2))
    rx, ry, back = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    rope_call(zkb, 0, [(x, rx)], b, n, d, d, False, freq, 1.0, pos, n, 0, False)
    rope_call(zkb, 0, [(rx, back)], b, n, d, d, False, freq, 1.0, pos, n, 0, True)
    rope_call(zkb, 0, [(y, ry)], b, n, d, d, False, freq, 1.0, pos, n, 0, True)
    size = x.abs() + x.abs().roll(d // 2, -1)
    near(back, x, torch.float32, 2 * ROPE_SLACK * 2 * size)
    dot = lambda u, v: (u.double() * v.double()).sum().item()  # noqa: E731
    assert abs(dot(rx, y) - dot(x, ry)) <= 4 * ROPE_SLACK * (size.double() * y.double().abs()).sum().item()


def test_rope_refuses_what_it_cannot_reach(zkb):
    z = zkb
    x = torch.zeros(1, 1, 1, 8, device="cuda")
    host = torch.zeros(1, 1, 1, 8)
    freq = rope_freq(8)

    def go(i, o, si=(8, 8, 8), so=(8, 8, 8), more=()):
        arr = z.rope_tensors((i, o, 1, si, so), *more)
        z.call("zkb_rope", 0, arr, 1 + len(more), 1, 1, 8, 8, 0, freq.data_ptr(), 1.0, None, 0, 0, 0, stream())
    p = x.data_ptr()
    for bad in ((host.data_ptr(), p), (p, host.data_ptr()), (p + 2, p), (None, p), (p, None)):
        with pytest.raises(z.ZkbError) as e:
            go(*bad)
        assert e.value.code == z.ERR_ARG
    with pytest.raises(z.ZkbError):
        go(p, p, so=(8, 16, 8))
    with pytest.raises(z.ZkbError):
        go(p, p, more=((p, p, 1, (8, 8, 8), (8, 8, 8)),))
    go(p, p)


# ---- norms --------------------------------------------------------------------------------------------------------------------------------


def norm_inputs(rows, cols, t, w, gate, post, seed, ld=None):
    g = gen(seed)
    ld = ld or cols
    mat = lambda by=1.0: (torch.randn(rows, ld, generator=g, device="cuda") * by).to(t)[:, :cols]  # noqa: E731
    vec = lambda: (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(w)  # noqa: E731
    gv = {"none": None, "channel": vec(), "row": torch.randn(rows, generator=g, device="cuda").to(t), "element": mat()}[gate]
    return mat(), mat(2.0), vec() if post else None, vec(), gv, mat(), mat()


def branch_of(y, post_gain, post, gate, kind, scale, eps):
    n = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() if post else y
    n = n * post_gain if post_gain is not None else n
    if gate is not None:
        n = n * (gate[:, None] if kind == "row" else gate)
    return scale * n


def wide(*xs):
    return [None if x is None else x.double() for x in xs]


def norm_call(z, code, wcode, x, y, post, post_gain, kind, gate, scale, pre_gain, eps, r, zz, post_inv, pre_inv, pre=1, st=None):
    rows, cols = x.shape
    z.call("zkb_block_norm", code, wcode, rows, cols, at(x), x.stride(0), at(y), y.stride(0) if y is not None else 0, int(post), at(post_gain),
           GATES.index(kind), at(gate), gate.stride(0) if kind == "element" else 0, scale, pre, at(pre_gain), eps, at(r), r.stride(0) if r is not None else 0, at(zz),
           zz.stride(0) if zz is not None else 0, at(post_inv), at(pre_inv), stream() if st is None else st)


def norm_slack(cols):
    """steps of 32 bits that a normed value may be off by: its statistics (a tree over cols squares, a quotient, a root: relative) and five products"""
    return (math.sqrt(cols) + 24) * F32


SIZES = [(1, 1), (3, 7), (5, 64), (2, 1000), (4, 1001), (17, 4096), (3, 5120), (2, 8192), (2, 8200), (3, 16384), (2, 16383), (300, 40)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,cols", SIZES)
def test_block_norm(zkb, kind, rows, cols):
    code, t = TYPES[kind]
    for i, gate in enumerate(GATES):
        post, w, wcode = i != 1, (t, torch.float32)[i % 2], (code, 0)[i % 2]
        x, y, pg, wg, gv, _, _ = norm_inputs(rows, cols, t, w, gate, post, rows + cols + i, ld=cols + (0, 8, 3, 0)[i])
        r, zz = torch.empty(rows, cols, device="cuda", dtype=t), torch.empty(rows, cols, device="cuda", dtype=t)
        pi, ri = (torch.empty(rows, device="cuda") for _ in range(2))
        norm_call(zkb, code, wcode, x, y, post, pg, gate, gv, 0.7, wg, 1e-5, r, zz, pi if post else None, ri)
        X, Y, PG, WG, GV = wide(x, y, pg, wg, gv)
        br = branch_of(Y, PG, post, GV, gate, 0.7, 1e-5)
        R = X + br
        rinv = 1 / (R.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
        k = norm_slack(cols)
        near(r, R, t, k * (X.abs() + br.abs()))
        near(zz, R * rinv * WG, t, 3 * k * (X.abs() + br.abs()) * rinv * WG.abs() + 3 * k * (R * rinv * WG).abs())
        near(ri, rinv[:, 0], torch.float32, 3 * k * rinv[:, 0])
        if post:
            near(pi, 1 / (Y.pow(2).mean(1) + 1e-5).sqrt(), torch.float32, k / (Y.pow(2).mean(1) + 1e-5).sqrt())


def test_block_norm_parts_alone_and_in_place(zkb):
    rows, cols, t = 33, 4096, torch.bfloat16
    x, y, pg, wg, gv, _, _ = norm_inputs(rows, cols, t, t, "element", True, 9)
    r, zz, both = torch.empty_like(x), torch.empty_like(x), []
    norm_call(zkb, 2, 2, x, y, True, pg, "element", gv, -0.5, wg, 1e-6, r, zz, None, None)
    # no branch: r is x, z its norm; unit gain
    z0, inv = torch.empty_like(x), torch.empty(rows, device="cuda")
    norm_call(zkb, 2, 2, x, None, False, None, "none", None, 1.0, None, 1e-6, None, z0, None, inv)
    near(z0, x.double() / (x.double().pow(2).mean(1, keepdim=True) + 1e-6).sqrt(), t, 3 * norm_slack(cols) * 6.0)
    # no norm before the next branch
    r1 = torch.empty_like(x)
    norm_call(zkb, 2, 2, x, y, True, pg, "element", gv, -0.5, None, 1e-6, r1, None, None, None, pre=0)
    assert torch.equal(r1, r)
    # statistics only
    inv2 = torch.empty(rows, device="cuda")
    norm_call(zkb, 2, 2, x, None, False, None, "none", None, 1.0, None, 1e-6, None, None, None, inv2)
    assert torch.equal(inv, inv2)
    # r over x, z over y
    x2, y2 = x.clone(), y.clone()
    norm_call(zkb, 2, 2, x2, y2, True, pg, "element", gv, -0.5, wg, 1e-6, x2, y2, None, None)
    assert torch.equal(x2, r) and torch.equal(y2, zz)


@pytest.mark.parametrize("kind", list(TYPES))
def test_block_norm_rows_that_hold_nothing_or_no_number(zkb, kind):
    """rows of zeros, of the type's largest values (their squares pass 32 bits for f32 and bf16: the norm is then zero, as in the formula with
    32-bit sums), with an infinity and with a NaN: each stays in its own row"""
    code, t = TYPES[kind]
    x = torch.randn(6, 100, generator=gen(1), device="cuda").to(t)
    clean = x.clone()
    x[1] = 0
    x[2] = torch.finfo(t).max
    x[3, 5] = math.inf
    x[4, 7] = math.nan
    out = {}
    for name, v in (("clean", clean), ("odd", x)):
        r, zz = torch.empty_like(x), torch.empty_like(x)
        norm_call(zkb, code, code, v, None, False, None, "none", None, 1.0, None, 1e-5, r, zz, None, None)
        out[name] = zz
    assert torch.equal(out["odd"][[0, 5]], out["clean"][[0, 5]])
    assert (out["odd"][1] == 0).all()
    assert torch.allclose(out["odd"][2].float(), torch.full((100,), 1.0 if kind == "f16" else 0.0, device="cuda"), atol=1e-3)
    assert out["odd"][3, 5].isnan() and (out["odd"][3].float().nan_to_num(0.0) == 0).all()
    assert out["odd"][4].isnan().all()


def norm_grads(x, y, pg, wg, gv, gate, post, scale, eps, dz, dr):
    """by torch's own differentiation of the formula in 64 bits; x is the stream before the branch"""
    leaves = {"x": x, "y": y, "pg": pg, "wg": wg, "gv": gv}
    v = {k: (u.detach().double().clone().requires_grad_(True) if u is not None else None) for k, u in leaves.items()}
    r = v["x"] + branch_of(v["y"], v["pg"], post, v["gv"], gate, scale, eps)
    zz = r / (r.pow(2).mean(-1, keepdim=True) + eps).sqrt() * v["wg"]
    loss = (zz * dz.double()).sum() + ((r * dr.double()).sum() if dr is not None else 0.0)
    used = {k: u for k, u in v.items() if u is not None}
    return dict(zip(used, torch.autograd.grad(loss, list(used.values())))), r.detach()


def back_call(z, code, wcode, r, y, post, pg, kind, gv, scale, wg, eps, dz, dr, dx, dy, dg, dpost, dpre, pre=1, st=None):
    rows, cols = (r if r is not None else y).shape
    s0 = lambda m: m.stride(0) if m is not None else 0  # noqa: E731
    el = kind == "element"
    z.call("zkb_block_norm_backward", code, wcode, rows, cols, at(r), s0(r), at(y), s0(y), int(post), at(pg), GATES.index(kind), at(gv), s0(gv) if el else 0, scale,
           pre, at(wg), eps, at(dz), s0(dz), at(dr), s0(dr), at(dx), s0(dx), at(dy), s0(dy), at(dg), s0(dg) if el else 0, at(dpost), at(dpre),
           stream() if st is None else st)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,cols", SIZES + [(700, 513)])
def test_block_norm_backward(zkb, kind, rows, cols):
    code, t = TYPES[kind]
    for i, gate in enumerate(GATES):
        post, w, wcode = i != 2, (t, torch.float32)[(i + 1) % 2], (code, 0)[(i + 1) % 2]
        r, y, pg, wg, gv, dz, dr = norm_inputs(rows, cols, t, w, gate, post, rows * 3 + cols + i, ld=cols + (3, 0, 8, 0)[i])
        dr = None if i == 1 else dr
        new = lambda *s, dtype=t: torch.full(s, math.nan, device="cuda", dtype=dtype)  # noqa: E731
        dx, dy, dpre, dpost = new(rows, cols), new(rows, cols), new(cols, dtype=w), new(cols, dtype=w) if post else None
        dg = {"none": None, "channel": new(cols, dtype=w), "row": new(rows), "element": new(rows, cols)}[gate]
        back_call(zkb, code, wcode, r, y, post, pg, gate, gv, 0.7, wg, 1e-5, dz, dr, dx, dy, dg, dpost, dpre)
        R, Y, PG, WG, GV = wide(r, y, pg, wg, gv)
        X = R - branch_of(Y, PG, post, GV, gate, 0.7, 1e-5)
        want, _ = norm_grads(X, y, pg, wg, gv, gate, post, 0.7, 1e-5, dz, dr)
        # sizes of the terms that make each gradient; each term is off by a few norm_slack of itself
        k = 8 * norm_slack(cols)
        rinv = 1 / (R.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
        p = (dz.double() * WG).abs()
        d = (dr.double().abs() if dr is not None else 0.0) + rinv * (p + R.abs() * rinv.pow(2) * (p * R.abs()).mean(1, keepdim=True))
        yinv = 1 / (Y.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() if post else torch.ones_like(rinv)
        gsize = 1.0 if GV is None else GV.abs()[:, None] if gate == "row" else GV.abs()
        dn = 0.7 * gsize * d
        q = dn * (PG.abs() if post else 1.0)
        dys = yinv * (q + (Y.abs() * yinv.pow(2) * (q * Y.abs()).mean(1, keepdim=True) if post else 0.0))
        near(dx, want["x"], t, k * d)
        near(dy, want["y"], t, k * dys)
        near(dpre, want["wg"], w, k * (dz.double() * R * rinv).abs().sum(0))
        if post:
            near(dpost, want["pg"], w, k * (dn * Y.abs() * yinv).sum(0))
        if GV is not None:
            each = 0.7 * d * (Y.abs() * yinv) * (PG.abs() if post else 1.0)
            each = {"channel": lambda: each.sum(0), "row": lambda: each.sum(1), "element": lambda: each}[gate]()
            near(dg, want["gv"], w if gate == "channel" else t, k * each)


def test_block_norm_backward_against_differences(zkb):
    """central differences of the forward formula in 64 bits, with one value of each input moved"""
    rows, cols, eps, h = 3, 24, 1e-3, 1e-6
    for gate in ("channel", "row", "element"):
        r, y, pg, wg, gv, dz, dr = norm_inputs(rows, cols, torch.float32, torch.float32, gate, True, 4)
        x = (r.double() - branch_of(*wide(y, pg), True, gv.double(), gate, 0.7, eps))
        out = {"x": torch.empty_like(r), "y": torch.empty_like(r), "gv": torch.empty_like(gv), "pg": torch.empty_like(pg), "wg": torch.empty_like(wg)}
        back_call(zkb, 0, 0, r, y, True, pg, gate, gv, 0.7, wg, eps, dz, dr, out["x"], out["y"], out["gv"], out["pg"], out["wg"])
        v = {"x": x, "y": y.double(), "pg": pg.double(), "wg": wg.double(), "gv": gv.double()}

        def loss(v):
            rr = v["x"] + branch_of(v["y"], v["pg"], True, v["gv"], gate, 0.7, eps)
            return ((rr / (rr.pow(2).mean(-1, keepdim=True) + eps).sqrt() * v["wg"]) * dz.double()).sum() + (rr * dr.double()).sum()
        for name in v:
            for place in (0, v[name].numel() - 1):
                up, down = ({k: u.clone() for k, u in v.items()} for _ in range(2))
                up[name].view(-1)[place] += h
                down[name].view(-1)[place] -= h
                slope = ((loss(up) - loss(down)) / (2 * h)).item()
                # the difference's own error is h^2 times a third derivative of order 100, and 2^-53 / h times the loss; the kernel's: 32 bits
                assert abs(out[name].view(-1)[place].item() - slope) <= 1e-5 * max(1.0, abs(slope)), (gate, name, place)


def test_block_norm_backward_parts(zkb):
    t = torch.float32
    r, y, pg, wg, gv, dz, dr = norm_inputs(50, 777, t, t, "channel", True, 12)
    full = [torch.empty_like(r), torch.empty_like(r), torch.empty_like(gv), torch.empty_like(pg), torch.empty_like(wg)]
    back_call(zkb, 0, 0, r, y, True, pg, "channel", gv, 0.7, wg, 1e-5, dz, dr, *full)
    for skip in range(5):     # any output left out changes no other
        part = [None if i == skip else torch.empty_like(o) for i, o in enumerate(full)]
        back_call(zkb, 0, 0, r, y, True, pg, "channel", gv, 0.7, wg, 1e-5, dz, dr, *part)
        assert all(p is None or torch.equal(p, o) for p, o in zip(part, full))
    # dx over dr, dy over y
    dr2, y2 = dr.clone(), y.clone()
    back_call(zkb, 0, 0, r, y2, True, pg, "channel", gv, 0.7, wg, 1e-5, dz, dr2, dr2, y2, None, None, None)
    assert torch.equal(dr2, full[0]) and torch.equal(y2, full[1])
    # no norm before the next branch: the gradient of r is what reaches it
    dx, dy = torch.empty_like(r), torch.empty_like(r)
    back_call(zkb, 0, 0, None, y, False, None, "channel", gv, 2.0, None, 1e-5, None, dr, dx, dy, None, None, None, pre=0)
    assert torch.equal(dx, dr) and torch.equal(dy, 2.0 * gv * dr)
    # no rows: zero sums
    z0 = [torch.ones(777, device="cuda") for _ in range(3)]
    zkb.call("zkb_block_norm_backward", 0, 0, 0, 777, at(r), 777, at(y), 777, 1, at(pg), 1, at(gv), 0, 0.7, 1, at(wg), 1e-5, at(dz), 777, None, 0, None, 0, None, 0,
             at(z0[0]), 0, at(z0[1]), at(z0[2]), stream())
    assert all((v == 0).all() for v in z0)


# ---- gated feed-forward ---------------------------------------------------------------------------------------------------------------------------


def act64(g, kind):
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
    if kind == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return g.clamp(min=0)


def glu_inputs(n, e, f, t, seed, pad=0, shift=0):
    g = gen(seed)

    def mat(r, c, by=1.0):
        buf = (torch.randn(r * (c + pad) + shift, generator=g, device="cuda") * by).to(t)
        return buf[shift:].view(r, c + pad)[:, :c]
    s = max(e, 1) ** -0.5
    return mat(n, e), mat(e, f, s), mat(e, f, s), mat(n, f), mat(n, f), mat(n, f)


def glu_call(z, code, act, x, wg, wu, h, gate, up, st=None):
    (n, e), f = x.shape, wg.shape[1]
    s0 = lambda m: 0 if m is None else m.stride(0)  # noqa: E731
    z.call("zkb_glu", code, ACTS.index(act), n, e, f, at(x), s0(x), at(wg), s0(wg), at(wu), s0(wu), at(h), s0(h), at(gate), s0(gate), at(up), s0(up),
           stream() if st is None else st)


def glu_back_call(z, code, act, x, wg, wu, gate, up, dh, dx, dwg, dwu, st=None):
    (n, e), f = x.shape, wg.shape[1]
    s0 = lambda m: 0 if m is None else m.stride(0)  # noqa: E731
    z.call("zkb_glu_backward", code, ACTS.index(act), n, e, f, at(x), s0(x), at(wg), s0(wg), at(wu), s0(wu), at(gate), s0(gate), at(up), s0(up), at(dh), s0(dh),
           at(dx), s0(dx), at(dwg), s0(dwg), at(dwu), s0(dwu), stream() if st is None else st)


def sum_slack(k):
    return (math.sqrt(k) + 8) * F32


def check_glu(z, kind, act, x, wg, wu, h, gate, up):
    t = TYPES[kind][1]
    X, G, U = wide(x, wg, wu)
    g, u = X @ G, X @ U
    ks = sum_slack(x.shape[1])
    eg, eu = ks * (X.abs() @ G.abs()), ks * (X.abs() @ U.abs())
    if gate is not None:
        near(gate, g, t, eg)
        near(up, u, t, eu)
    # |act'| <= 1.2 for all four; the activation itself is formed to 2^-20 of |g| (a fast exponential of a bounded argument)
    a = act64(g, act)
    near(h, a * u, t, (1.2 * eg + 2.0 ** -20 * (g.abs() + eg)) * (u.abs() + eu) + a.abs() * eu)


GLU_SIZES = [(1, 1, 1), (1, 64, 128), (3, 65, 127), (5, 8, 8), (16, 256, 512), (17, 130, 70), (1, 4096, 264), (33, 1000, 136), (64, 96, 200), (65, 512, 384),
             (127, 129, 131), (128, 128, 128), (129, 200, 520), (300, 264, 777), (513, 72, 1032), (8, 2056, 3000)]


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("n,e,f", GLU_SIZES)
def test_glu(zkb, kind, n, e, f):
    code, t = TYPES[kind]
    for i, (pad, shift) in enumerate(((0, 0), (8, 0), (5, 3))):
        act = ACTS[(n + e + f + i) % 4]
        x, wg, wu, _, _, _ = glu_inputs(n, e, f, t, n + e + f + i, pad, shift)
        guard = torch.full((n + 2, f + pad + 1), 5.0, device="cuda", dtype=t)
        h = guard[1:n + 1, :f]
        keep = [torch.empty(n, f, device="cuda", dtype=t) for _ in range(2)] if i != 1 else [None, None]
        glu_call(zkb, code, act, x, wg, wu, h, *keep)
        check_glu(zkb, kind, act, x, wg, wu, h, *keep)
        assert (guard[0] == 5).all() and (guard[n + 1] == 5).all() and (guard[:, f:] == 5).all()   # rows and columns around stay as they were
        again = torch.empty_like(h)
        glu_call(zkb, code, act, x, wg, wu, again, *keep)
        assert torch.equal(again, h)


def test_glu_without_inputs(zkb):
    h = torch.full((3, 5), 9.0, device="cuda", dtype=torch.bfloat16)
    zkb.call("zkb_glu", 2, 0, 3, 0, 5, None, 0, None, 0, None, 0, at(h), 5, None, 0, None, 0, stream())
    assert (h == 0).all()


@pytest.mark.parametrize("act", ACTS)
def test_glu_far_and_missing_values(zkb, act):
    """an activation far from zero, an infinity and a NaN in one token each: the others' results stay"""
    n, e, f = 140, 128, 192
    x, wg, wu, _, _, _ = glu_inputs(n, e, f, torch.bfloat16, 77)
    h0, h1 = torch.empty(n, f, device="cuda", dtype=torch.bfloat16), torch.empty(n, f, device="cuda", dtype=torch.bfloat16)
    glu_call(zkb, 2, act, x, wg, wu, h0, None, None)
    x = x.clone()
    x[3] *= 1000
    x[70, 1] = math.inf
    x[139, 0] = math.nan
    glu_call(zkb, 2, act, x, wg, wu, h1, None, None)
    same = torch.ones(n, dtype=torch.bool, device="cuda")
    same[[3, 70, 139]] = False
    assert torch.equal(h1[same], h0[same])
    check_glu(zkb, "bf16", act, x[3:4], wg, wu, h1[3:4], None, None)
    assert h1[139].isnan().all() and not h1[70].isfinite().any() or act == "relu"


def glu_grads(act, x, wg, wu, gate, up, dh):
    g, u = (v.double().requires_grad_(True) for v in (gate, up))
    dg, du = torch.autograd.grad((act64(g, act) * u * dh.double()).sum(), (g, u))
    X, G, U = wide(x, wg, wu)
    return dg, du, dg @ G.T + du @ U.T, X.T @ dg, X.T @ du


def check_glu_back(z, kind, act, x, wg, wu, gate, up, dh, dx, dwg, dwu):
    t = TYPES[kind][1]
    n, e = x.shape
    dg, du, wx, wgg, wgu = glu_grads(act, x, wg, wu, gate, up, dh)
    X, G, U, D, UP, GT = wide(x, wg, wu, dh, up, gate)
    # each projection's gradient is off by half a step when it is rounded, and before that by 2^-20 of its factors' size (fast exponential)
    eg = half_step(t) * dg.abs() + 2.0 ** -19 * (D * UP).abs() * (1 + GT.abs()) + tiny(t)
    eu = half_step(t) * du.abs() + 2.0 ** -20 * (D * GT).abs() + tiny(t)
    if dx is not None:
        near(dx, wx, t, eg @ G.abs().T + eu @ U.abs().T + sum_slack(2 * wg.shape[1]) * (dg.abs() @ G.abs().T + du.abs() @ U.abs().T))
    if dwg is not None:
        near(dwg, wgg, t, X.abs().T @ eg + sum_slack(n) * (X.abs().T @ dg.abs()))
        near(dwu, wgu, t, X.abs().T @ eu + sum_slack(n) * (X.abs().T @ du.abs()))


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("n,e,f", GLU_SIZES)
def test_glu_backward(zkb, kind, n, e, f):
    code, t = TYPES[kind]
    for i, (pad, shift) in enumerate(((0, 0), (8, 0), (5, 3))):
        act = ACTS[(n + e + f + i) % 4]
        x, wg, wu, gate, up, dh = glu_inputs(n, e, f, t, n * 2 + e + f + i, pad, shift)
        guard = torch.full((n + 2, e + pad + 1), 5.0, device="cuda", dtype=t)
        wguard = torch.full((e + 2, f + pad + 1), 5.0, device="cuda", dtype=t)
        dx, dwg, dwu = guard[1:n + 1, :e], wguard[1:e + 1, :f], torch.full((e, f), math.nan, device="cuda", dtype=t)
        glu_back_call(zkb, code, act, x, wg, wu, gate, up, dh, dx, dwg, dwu)
        check_glu_back(zkb, kind, act, x, wg, wu, gate, up, dh, dx, dwg, dwu)
        for gd, k in ((guard, n), (wguard, e)):
            assert (gd[0] == 5).all() and (gd[k + 1] == 5).all()
        assert (guard[:, e:] == 5).all() and (wguard[:, f:] == 5).all()
        if i == 0:     # each result alone, and the same bits again
            dx2, dwg2, dwu2 = torch.empty_like(dx), torch.empty_like(dwg), torch.empty_like(dwu)
            glu_back_call(zkb, code, act, x, wg, wu, gate, up, dh, dx2, None, None)
            glu_back_call(zkb, code, act, x, wg, wu, gate, up, dh, None, dwg2, dwu2)
            assert torch.equal(dx2, dx) and torch.equal(dwg2, dwg) and torch.equal(dwu2, dwu)


def test_glu_backward_of_no_tokens_and_no_channels(zkb):
    t = torch.float16
    w = torch.ones(4, 6, device="cuda", dtype=t)
    dwg, dwu, dx = torch.ones_like(w), torch.ones_like(w), torch.ones(3, 4, device="cuda", dtype=t)
    zkb.call("zkb_glu_backward", 1, 0, 0, 4, 6, None, 4, at(w), 6, at(w), 6, None, 6, None, 6, None, 6, None, 4, at(dwg), 6, at(dwu), 6, stream())
    assert (dwg == 0).all() and (dwu == 0).all()
    zkb.call("zkb_glu_backward", 1, 0, 3, 4, 0, at(dx), 4, None, 0, None, 0, None, 0, None, 0, None, 0, at(dx), 4, None, 0, None, 0, stream())
    assert (dx == 0).all()


def test_glu_backward_against_differences(zkb):
    """central differences of the block in 64 bits; the kept projections are the ones of the forward call, rounded: f16 gradients agree to the
    rounding of what goes into them (a few steps of 2^-11 of the terms' sum)"""
    n, e, f, h = 4, 16, 24, 1e-5
    for act in ACTS[:3]:
        x, wg, wu, _, _, dh = glu_inputs(n, e, f, torch.float16, 21)
        hh, gate, up = (torch.empty(n, f, device="cuda", dtype=torch.float16) for _ in range(3))
        glu_call(zkb, 1, act, x, wg, wu, hh, gate, up)
        out = {"x": torch.empty_like(x), "wg": torch.empty_like(wg), "wu": torch.empty_like(wu)}
        glu_back_call(zkb, 1, act, x, wg, wu, gate, up, dh, out["x"], out["wg"], out["wu"])
        v = {"x": x.double(), "wg": wg.double(), "wu": wu.double()}
        loss = lambda v: (act64(v["x"] @ v["wg"], act) * (v["x"] @ v["wu"]) * dh.double()).sum()  # noqa: E731
        dg, du, _, _, _ = glu_grads(act, x, wg, wu, gate, up, dh)
        size = {"x": dg.abs() @ v["wg"].abs().T + du.abs() @ v["wu"].abs().T, "wg": v["x"].abs().T @ dg.abs(), "wu": v["x"].abs().T @ du.abs()}
        # rounding gate and up moves dg by its second derivative (below 2) times their half steps: 2 h |dh u| (1 + |g|) more
        extra = 2 * 2.0 ** -11 * (dh.double().abs() * (up.double().abs() + 1) * (1 + gate.double().abs()))
        size = {"x": size["x"] * 2.0 ** -10 + extra @ (v["wg"].abs() + v["wu"].abs()).T, "wg": size["wg"] * 2.0 ** -10 + v["x"].abs().T @ extra,
                "wu": size["wu"] * 2.0 ** -10 + v["x"].abs().T @ extra}
        for name in v:
            for place in (0, 7, v[name].numel() - 1):
                a, b = ({k: u.clone() for k, u in v.items()} for _ in range(2))
                a[name].view(-1)[place] += h
                b[name].view(-1)[place] -= h
                slope = ((loss(a) - loss(b)) / (2 * h)).item()
                assert abs(out[name].view(-1)[place].item() - slope) <= size[name].view(-1)[place].item() + 1e-5, (act, name, place)


def test_glu_refuses_what_it_cannot_reach(zkb):
    z = zkb
    t = torch.bfloat16
    x, wg, wu, gate, up, dh = glu_inputs(2, 8, 8, t, 1)
    h, host = torch.empty(2, 8, device="cuda", dtype=t), torch.empty(8, 8, dtype=t)
    for bad in ((host[:2], wg, wu, h), (x, host, wu, h), (x, wg, host, h), (x, wg, wu, host[:2])):
        with pytest.raises(z.ZkbError) as e:
            glu_call(z, 2, "silu", *bad, None, None)
        assert e.value.code == z.ERR_ARG
    with pytest.raises(z.ZkbError):
        z.call("zkb_glu", 2, 0, 2, 8, 8, at(x) + 1, 8, at(wg), 8, at(wu), 8, at(h), 8, None, 0, None, 0, stream())
    with pytest.raises(z.ZkbError):
        norm_call(z, 2, 2, host, None, False, None, "none", None, 1.0, None, 1e-5, None, None, None, None)


# ---- together, streams, graphs ------------------------------------------------------------------------------------------------------------------


class Layer:
    """One decoder layer's float pass and its gradients, with attention itself in torch: norm, rotary positions, the norms around both branches
    and the feed-forward block through the library; `plain` computes the same in 64 bits by torch alone."""

    def __init__(self, z, n, heads, d, f, seed):
        self.z, self.n, self.heads, self.d, self.f = z, n, heads, d, f
        e = heads * d
        g = gen(seed)
        t = torch.float16
        rnd = lambda *s, by=1.0: (torch.randn(*s, generator=g, device="cuda") * by).to(t)  # noqa: E731
        self.x = rnd(n, e)
        self.w = {k: rnd(*s, by=s[0] ** -0.5) for k, s in {"q": (e, e), "k": (e, e), "v": (e, e), "wg": (e, f), "wu": (e, f), "down": (f, e)}.items()}
        self.gain = {k: (1 + 0.1 * torch.randn(e, generator=g, device="cuda")).to(t) for k in ("in", "post", "mid", "post2")}
        self.freq, self.pos = rope_freq(d), torch.arange(n, device="cuda") + 11
        self.t, self.e = t, e
        self.buf = {k: torch.empty(n, e, device="cuda", dtype=t) for k in ("h0", "r1", "h1", "r2")}
        self.qr, self.kr = (torch.empty(1, n, heads, d, device="cuda", dtype=t) for _ in range(2))
        self.h, self.g, self.u = (torch.empty(n, f, device="cuda", dtype=t) for _ in range(3))

    def run(self):
        z, b, w, gn, n = self.z, self.buf, self.w, self.gain, self.n
        norm_call(z, 1, 1, self.x, None, False, None, "none", None, 1.0, gn["in"], 1e-5, None, b["h0"], None, None)
        q, k, v = ((b["h0"] @ w[c]).view(1, n, self.heads, self.d) for c in "qkv")
        rope_call(z, 1, [(q, self.qr), (k, self.kr)], 1, n, self.d, self.d, False, self.freq, 1.0, self.pos, n, 0, False)
        s = torch.einsum("bthd,bshd->bhts", self.qr.float(), self.kr.float()) * self.d ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf).softmax(-1)
        self.att = torch.einsum("bhts,bshd->bthd", s, v.float()).reshape(n, self.e).to(self.t)
        norm_call(z, 1, 1, self.x, self.att, True, gn["post"], "none", None, 0.5, gn["mid"], 1e-5, b["r1"], b["h1"], None, None)
        glu_call(z, 1, "silu", b["h1"], w["wg"], w["wu"], self.h, self.g, self.u)
        self.ffn = self.h @ w["down"]
        norm_call(z, 1, 1, b["r1"], self.ffn, True, gn["post2"], "none", None, 0.5, None, 1e-5, b["r2"], None, None, None, pre=0)
        return b["r2"]

    def plain(self):
        d = lambda x: x.double()  # noqa: E731
        nrm = lambda v, w: v / (v.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * d(w)  # noqa: E731
        h0 = nrm(d(self.x), self.gain["in"])
        q, k, v = ((h0 @ d(self.w[c])).view(1, self.n, self.heads, self.d) for c in "qkv")
        q, k = (rope_want(x, self.pos[None], self.freq, 1.0, self.d, False, False)[0] for x in (q, k))
        s = torch.einsum("bthd,bshd->bhts", q, k) * self.d ** -0.5
        s = s.masked_fill(torch.ones(self.n, self.n, dtype=torch.bool, device="cuda").triu(1), -math.inf).softmax(-1)
        att = torch.einsum("bhts,bshd->bthd", s, v).reshape(self.n, self.e)
        r1 = d(self.x) + 0.5 * nrm(att, self.gain["post"])
        h1 = nrm(r1, self.gain["mid"])
        ffn = (act64(h1 @ d(self.w["wg"]), "silu") * (h1 @ d(self.w["wu"]))) @ d(self.w["down"])
        return r1 + 0.5 * nrm(ffn, self.gain["post2"])


def test_a_layer_of_them(zkb):
    """about ten roundings to f16 lie between the input and the result, each off by 2^-11 of its value at most and 2^-13 in the mean square; through
    norms and sums they add up like independent errors to well below 2^-9 of the result's norm"""
    layer = Layer(zkb, 150, 4, 32, 328, 8)
    got, want = layer.run().double(), layer.plain()
    assert ((got - want).norm() / want.norm()).item() < 2.0 ** -9


@pytest.mark.parametrize("what", ("layer", "backward"))
def test_captured_graphs_replay_side_by_side(zkb, what):
    """two graphs of the same calls on data of their own, replayed on two streams at once, again after their inputs changed"""
    def make(seed):
        if what == "layer":
            layer = Layer(zkb, 70, 2, 32, 136, seed)
            return layer.x, lambda: [layer.run()]
        t = torch.bfloat16
        x, wg, wu, gate, up, dh = glu_inputs(200, 136, 328, t, seed)
        r, y, pg, gg, gv, dz, dr = norm_inputs(300, 520, t, t, "channel", True, seed)
        outs = [torch.empty(200, 136, device="cuda", dtype=t), torch.empty(136, 328, device="cuda", dtype=t), torch.empty(136, 328, device="cuda", dtype=t)]
        nouts = [torch.empty_like(r), torch.empty_like(r), torch.empty_like(gv), torch.empty_like(pg), torch.empty_like(gg)]

        def go():
            glu_back_call(zkb, 2, "silu", x, wg, wu, gate, up, dh, *outs)
            back_call(zkb, 2, 2, r, y, True, pg, "channel", gv, 0.7, gg, 1e-5, dz, dr, *nouts)
            return outs + nouts
        return dh, go
    torch.cuda.synchronize()
    made = [make(s) for s in (1, 2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in made]
    for (_, go), st in zip(made, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            go()                        # libraries that torch itself calls set up here
        st.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            res = go()
        graphs.append((gr, res))
    torch.cuda.synchronize()
    for turn in range(3):
        for x, _ in made:
            x.mul_(-0.5)
        torch.cuda.synchronize()
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        replayed = [[o.clone() for o in res] for _, res in graphs]
        eager = [[o.clone() for o in go()] for _, go in made]
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
    del graphs


def test_another_stream_orders_its_own_work(zkb):
    """calls on a stream of the library's own making, beside others on torch's"""
    z = zkb
    st = ctypes.c_void_p()
    z.call("zkb_stream_create", ctypes.c_int(1), ctypes.byref(st))
    t = torch.bfloat16
    x, wg, wu, gate, up, dh = glu_inputs(130, 264, 520, t, 5)
    a, b = torch.empty(130, 520, device="cuda", dtype=t), torch.empty(130, 520, device="cuda", dtype=t)
    torch.cuda.synchronize()
    for _ in range(5):
        glu_call(z, 2, "silu", x, wg, wu, a, None, None, st=st.value)
        glu_call(z, 2, "silu", x, wg, wu, b, None, None)
    z.call("zkb_sync", z._p(st.value))
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    check_glu(z, "bf16", "silu", x, wg, wu, a, None, None)
    z.call("zkb_stream_destroy", z._p(st.value))


@pytest.mark.skipif(torch.cuda.is_available() and torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_devices_memory_is_refused(zkb):
    x = torch.zeros(2, 8, device="cuda:1")
    with pytest.raises(zkb.ZkbError) as e:
        norm_call(zkb, 0, 0, x, None, False, None, "none", None, 1.0, None, 1e-5, None, torch.zeros(2, 8, device="cuda:0"), None, None, st=0)
    assert e.value.code == zkb.ERR_ARG


def test_pinned_host_memory_is_refused(zkb):
    x = torch.zeros(2, 8).pin_memory()
    out = torch.zeros(2, 8, device="cuda")
    with pytest.raises(zkb.ZkbError) as e:
        norm_call(zkb, 0, 0, x, None, False, None, "none", None, 1.0, None, 1e-5, None, out, None, None)
    assert e.value.code == zkb.ERR_ARG


@pytest.mark.parametrize("n,e,f", [(4400, 72, 1100), (2560, 2048, 264), (2700, 1800, 520)])
def test_glu_many_tiles(zkb, n, e, f):
    """more rows of tiles than a band holds; more long tiles of dx than pairs of blocks, beside short ones of the weights"""
    t = torch.bfloat16
    x, wg, wu, gate, up, dh = glu_inputs(n, e, f, t, n)
    h, g, u = (torch.empty(n, f, device="cuda", dtype=t) for _ in range(3))
    glu_call(zkb, 2, "gelu", x, wg, wu, h, g, u)
    check_glu(zkb, "bf16", "gelu", x, wg, wu, h, g, u)
    dx, dwg, dwu = torch.full_like(x, math.nan), torch.full_like(wg, math.nan), torch.full_like(wu, math.nan)
    glu_back_call(zkb, 2, "gelu", x, wg, wu, gate, up, dh, dx, dwg, dwu)
    check_glu_back(zkb, "bf16", "gelu", x, wg, wu, gate, up, dh, dx, dwg, dwu)


@pytest.mark.parametrize("rows,cols", [(5000, 96), (700, 4100), (310, 6000), (200, 12000), (160, 16384)])
def test_block_norm_many_rows(zkb, rows, cols):
    """more rows than resident blocks times slots, in each of the kernels' layouts, aligned and not: the ring goes round"""
    for t, code, shift in ((torch.bfloat16, 2, 0), (torch.float32, 0, 0), (torch.float16, 1, 1)):
        if cols + shift > 16384:     # refused: beyond the documented limit
            continue
        r, y, pg, wg, gv, dz, dr = norm_inputs(rows, cols + shift, t, t, "element", True, rows + cols)
        x = r
        ro, zz, inv = torch.empty(rows, cols + shift, device="cuda", dtype=t), torch.empty(rows, cols + shift, device="cuda", dtype=t), torch.empty(rows, device="cuda")
        norm_call(zkb, code, code, x, y, True, pg, "element", gv, 0.7, wg, 1e-5, ro, zz, None, inv)
        X, Y, PG, WG, GV = wide(x, y, pg, wg, gv)
        br = branch_of(Y, PG, True, GV, "element", 0.7, 1e-5)
        R = X + br
        rinv = 1 / (R.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
        k = norm_slack(cols + shift)
        near(ro, R, t, k * (X.abs() + br.abs()))
        near(zz, R * rinv * WG, t, 3 * k * (X.abs() + br.abs()) * rinv * WG.abs() + 3 * k * (R * rinv * WG).abs())
        near(inv, rinv[:, 0], torch.float32, 3 * k * rinv[:, 0])
        outs = [torch.full_like(r, math.nan), torch.full_like(y, math.nan), torch.full_like(gv, math.nan), torch.full_like(pg, math.nan), torch.full_like(wg, math.nan)]
        back_call(zkb, code, code, r, y, True, pg, "element", gv, 0.7, wg, 1e-5, dz, dr, *outs)
        want, _ = norm_grads(X - br, y, pg, wg, gv, "element", True, 0.7, 1e-5, dz, dr)   # the stream before the branch, so that r is the sum
        R = X
        rinv = 1 / (R.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
        p = (dz.double() * WG).abs()
        d = dr.double().abs() + rinv * (p + R.abs() * rinv.pow(2) * (p * R.abs()).mean(1, keepdim=True))
        yinv = 1 / (Y.pow(2).mean(1, keepdim=True) + 1e-5).sqrt()
        q = 0.7 * GV.abs() * d * PG.abs()
        near(outs[0], want["x"], t, 8 * k * d)
        near(outs[1], want["y"], t, 8 * k * yinv * (q + Y.abs() * yinv.pow(2) * (q * Y.abs()).mean(1, keepdim=True)))
        near(outs[2], want["gv"], t, 8 * k * 0.7 * d * Y.abs() * yinv * PG.abs())
        near(outs[3], want["pg"], t, 8 * norm_slack(rows + cols) * (0.7 * GV.abs() * d * Y.abs() * yinv).sum(0))
        near(outs[4], want["wg"], t, 8 * norm_slack(rows + cols) * (dz.double() * R * rinv).abs().sum(0))
        again = [torch.empty_like(o) for o in outs]
        back_call(zkb, code, code, r, y, True, pg, "element", gv, 0.7, wg, 1e-5, dz, dr, *again)
        assert all(torch.equal(a, b) for a, b in zip(again, outs))


def test_two_host_threads_at_once(zkb):
    """calls of two threads on streams and data of their own, interleaved as they come"""
    import threading
    t = torch.bfloat16
    sets, errors = [], []
    for seed in (1, 2):
        x, wg, wu, gate, up, dh = glu_inputs(150, 264, 520, t, seed)
        r, y, pg, gg, gv, dz, dr = norm_inputs(600, 1032, t, t, "channel", True, seed)
        outs = [torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)]
        nouts = [torch.empty_like(r), torch.empty_like(r), torch.empty_like(gv), torch.empty_like(pg), torch.empty_like(gg)]
        h = torch.empty(9, 520, device="cuda", dtype=t)
        sets.append((x, wg, wu, gate, up, dh, r, y, pg, gg, gv, dz, dr, outs, nouts, h))

    def once(s, st):
        x, wg, wu, gate, up, dh, r, y, pg, gg, gv, dz, dr, outs, nouts, h = s
        glu_back_call(zkb, 2, "silu", x, wg, wu, gate, up, dh, *outs, st=st)
        back_call(zkb, 2, 2, r, y, True, pg, "channel", gv, 0.7, gg, 1e-5, dz, dr, *nouts, st=st)
        glu_call(zkb, 2, "silu", x[:9], wg, wu, h, None, None, st=st)
    for s in sets:
        once(s, stream())
    torch.cuda.synchronize()
    want = [[o.clone() for o in s[13] + s[14] + [s[15]]] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]

    def work(s, st):
        try:
            torch.cuda.set_device(0)
            for _ in range(30):
                once(s, st.cuda_stream)
            st.synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=a) for a in zip(sets, streams)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(s[13] + s[14] + [s[15]], w))


def test_a_capture_may_hold_the_first_call(tmp_path):
    """in a process of its own, the first call of each operator is made while its stream is captured"""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    code = """
import sys
sys.path.insert(0, {root!r})
import torch
from tests import test_gpu_floatops as T
from tests.conftest import load_package
z = load_package()
t = torch.bfloat16
x, wg, wu, gate, up, dh = T.glu_inputs(200, 136, 328, t, 1)
r, y, pg, gg, gv, dz, dr = T.norm_inputs(300, 520, t, t, "channel", True, 1)
h, h9 = torch.zeros(200, 328, device="cuda", dtype=t), torch.zeros(9, 328, device="cuda", dtype=t)
outs = [torch.zeros_like(x), torch.zeros_like(wg), torch.zeros_like(wu)]
nouts = [torch.zeros_like(r), torch.zeros_like(r), torch.zeros_like(gv), torch.zeros_like(pg), torch.zeros_like(gg)]
zz, rr = torch.zeros_like(r), torch.zeros_like(r)
q = torch.randn(1, 200, 2, 64, device="cuda", dtype=t)
qo, freq = torch.zeros_like(q), T.rope_freq(64)
def go():
    T.glu_call(z, 2, "silu", x, wg, wu, h, None, None)
    T.glu_call(z, 2, "silu", x[:9], wg, wu, h9, None, None)
    T.glu_back_call(z, 2, "silu", x, wg, wu, gate, up, dh, *outs)
    T.norm_call(z, 2, 2, r, y, True, pg, "channel", gv, 0.7, gg, 1e-5, rr, zz, None, None)
    T.back_call(z, 2, 2, r, y, True, pg, "channel", gv, 0.7, gg, 1e-5, dz, dr, *nouts)
    T.rope_call(z, 2, [(q, qo)], 1, 200, 64, 64, False, freq, 1.0, None, 0, 5, False)
torch.cuda.synchronize()
g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(g, stream=st):
    go()
everything = [h, h9, rr, zz, qo] + outs + nouts
g.replay()
torch.cuda.synchronize()
first = [o.clone() for o in everything]
go()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first, everything)) and all(a.any() for a in first)
print("same")
""".format(root=str(root))
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=root)
    assert res.returncode == 0 and "same" in res.stdout, res.stdout[-1000:] + res.stderr[-3000:]


def test_the_rms_inv_stage_feeds_rmsnorm(tmp_path):
    """the driver's rms-inv stage writes what the rmsnorm stage reads: within one unit of the formula in 64 bits (32-bit statistics of values of
    2^16 are off by less than 2^-20 of themselves, a sixteenth of a unit, which moves a rounding now and then); then rmsnorm proves with it, in
    one batch"""
    import numpy as np
    from tests.test_gpu_drivers import BIN, make_param, rescale, run, save_int
    rng = np.random.Generator(np.random.PCG64(5))
    seq, embed = 256, 256
    x = np.rint(rng.standard_normal((seq, embed)) * 65536 * np.exp(rng.standard_normal((seq, 1)))).astype(np.int64)
    w = np.rint((1.0 + 0.1 * rng.standard_normal(embed)) * 65536).astype(np.int64)
    save_int(tmp_path / "x.bin", x)
    make_param(BIN, tmp_path, "layer-0", "input_layernorm.weight", w, 1, embed, embed)
    (tmp_path / "script").write_text(f"rms-inv x.bin {seq} {embed} 1e-5\nrmsnorm input x.bin {seq} {embed} {tmp_path} layer-0 out.bin\n")
    run(BIN, "zkllm-driver", ["batch", "script"], tmp_path)
    got = np.fromfile(tmp_path / "rms_inv_temp.bin", dtype=np.int32).astype(np.int64)
    want = 65536.0 / np.sqrt(((x / 65536.0) ** 2).mean(axis=1) + 1e-5)
    assert got.shape == (seq,) and np.abs(got - want).max() <= 0.5 + 2.0 ** -20 * want.max()
    exp = rescale(rescale(np.outer(got, w), 1 << 16) * x, 1 << 16)
    assert np.array_equal(np.fromfile(tmp_path / "out.bin", dtype=np.int32).astype(np.int64), exp.reshape(-1))
    import subprocess
    for bad in (["x.bin", seq, embed + 1, 1e-5], ["x.bin", seq, embed, 0.0]):
        res = subprocess.run([str(BIN / "zkllm-driver"), "rms-inv", *map(str, bad)], cwd=tmp_path, capture_output=True, text=True, timeout=120)
        assert res.returncode != 0


def test_a_call_waits_for_the_one_before(zkb):
    """each kind of call takes what the one before it on the stream has just written, many rows of it, with nothing between: norm to few tokens, few
    tokens to norm, norm to norm, gradients of the norm to few tokens, few tokens to few tokens in the same workspace"""
    t, n, e, f = torch.bfloat16, 6000, 1024, 1536
    x, wg, wu, _, _, _ = glu_inputs(n, e, f, t, 3)
    r, y, pg, gg, gv, dz, dr = norm_inputs(n, e, t, t, "channel", True, 3)
    z1, z2, dx, dy = (torch.empty(n, e, device="cuda", dtype=t) for _ in range(4))
    last = slice(n - 16, n)
    h = [torch.empty(16, f, device="cuda", dtype=t) for _ in range(4)]
    zh = torch.empty(16, f, device="cuda", dtype=t)
    dg, dp, dw = torch.empty_like(gv), torch.empty_like(pg), torch.empty_like(gg)

    def chain(pause):
        for o in [z1, z2, dx, dy, zh, dg, dp, dw] + h:
            o.zero_()
        pause()
        norm_call(zkb, 2, 2, x, None, False, None, "none", None, 1.0, gg, 1e-5, None, z1, None, None)
        pause()
        glu_call(zkb, 2, "silu", z1[last], wg, wu, h[0], None, None)
        pause()
        norm_call(zkb, 2, 2, h[0], None, False, None, "none", None, 1.0, None, 1e-5, None, zh, None, None)
        pause()
        norm_call(zkb, 2, 2, z1, y, True, pg, "channel", gv, 0.7, gg, 1e-5, None, z2, None, None)
        pause()
        glu_call(zkb, 2, "silu", z2[last], wg, wu, h[1], None, None)
        pause()
        glu_call(zkb, 2, "gelu", z1[last], wg, wu, h[2], None, None)
        pause()
        back_call(zkb, 2, 2, z2, y, True, pg, "channel", gv, 0.7, gg, 1e-5, dz, dr, dx, dy, dg, dp, dw)
        pause()
        glu_call(zkb, 2, "silu", dx[last], wg, wu, h[3], None, None)
        torch.cuda.synchronize()
        return [o.clone() for o in [z1, z2, dx, dy, zh, dg, dp, dw] + h]
    want = chain(torch.cuda.synchronize)
    for _ in range(20):
        got = chain(lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
