"""GPU: the float operators of a layer where a type's range, a wait or a neighbouring call could spoil a result.

Tolerances as in test_gpu_floatops.py: half a step of the type for each rounding, and for the 32-bit arithmetic before it what each test derives."""
import ctypes
import math
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests.test_gpu_floatops import (  # noqa: E402
    ACTS, TYPES, back_call, glu_back_call, glu_call, glu_grads, glu_inputs, half_step, near, norm_call, norm_inputs, rope_call, rope_freq, stream,
    sum_slack, wide)


# ---- gradients of the feed-forward block in f16 --------------------------------------------------------------------------------------------


def check_scaled(act, x, wg, wu, gate, up, dh, dx, dwg, dwu, rows=slice(None)):
    """The gradients of the projections are rounded to f16 at a scale that puts the call's largest at 2^14 or above: each is off by half a step of
    its value or by 2^-25 at that scale, 2^-39 of the largest, and before that by 2^-19 of its factors' size (fast exponential)."""
    t = torch.float16
    dg, du, wx, wgg, wgu = glu_grads(act, x, wg, wu, gate, up, dh)
    X, G, U, D, UP, GT = wide(x, wg, wu, dh, up, gate)
    peak = torch.maximum(dg.abs().max(), du.abs().max())
    eg = half_step(t) * dg.abs() + 2.0 ** -19 * (D * UP).abs() * (1 + GT.abs()) + 2.0 ** -39 * peak
    eu = half_step(t) * du.abs() + 2.0 ** -20 * (D * GT).abs() + 2.0 ** -39 * peak
    near(dx[rows], wx[rows], t, (eg @ G.abs().T + eu @ U.abs().T + sum_slack(2 * wg.shape[1]) * (dg.abs() @ G.abs().T + du.abs() @ U.abs().T))[rows])
    if dwg is None:
        return
    near(dwg, wgg, t, X.abs().T @ eg + sum_slack(x.shape[0]) * (X.abs().T @ dg.abs()))
    near(dwu, wgu, t, X.abs().T @ eu + sum_slack(x.shape[0]) * (X.abs().T @ du.abs()))
    # the roundings are independent: relative to a result's norm they make half a step together, and the result's own another
    for got, want in ((dx, wx), (dwg, wgg), (dwu, wgu)):
        assert ((got.double() - want).norm() / want.norm()).item() <= 2.0 ** -10


# sizes of dh, of up and gate, of x and of the weights: products far below f16's normal numbers and above its largest, results that f16 holds well
@pytest.mark.parametrize("by", [(1e-5, 1.0, 64.0, 64.0), (1e-6, 1.0, 512.0, 1024.0), (2.0 ** -21, 0.05, 8192.0, 32768.0), (300.0, 300.0, 2.0 ** -9, 2.0 ** -8),
                                (10000.0, 0.5, 2.0 ** -6, 2.0 ** -6)])
@pytest.mark.parametrize("n,e,f,pad,shift", [(513, 72, 1032, 0, 0), (40, 264, 520, 5, 3), (777, 520, 136, 0, 0)])
def test_glu_backward_f16_of_small_and_large_gradients(zkb, n, e, f, pad, shift, by):
    for act in ACTS:
        x, wg, wu, gate, up, dh = glu_inputs(n, e, f, torch.float16, n + e, pad, shift)
        for m, k in ((dh, by[0]), (up, by[1]), (x, by[2]), (wg, by[3]), (wu, by[3])):
            m.mul_(k)
        if by[1] < 1:
            gate.mul_(by[1])
        dx, dwg, dwu = torch.full_like(x, math.nan), torch.full_like(wg, math.nan), torch.full_like(wu, math.nan)
        glu_back_call(zkb, 1, act, x, wg, wu, gate, up, dh, dx, dwg, dwu)
        check_scaled(act, x, wg, wu, gate, up, dh, dx, dwg, dwu)
        again = [torch.empty_like(o) for o in (dx, dwg, dwu)]
        glu_back_call(zkb, 1, act, x, wg, wu, gate, up, dh, *again)
        assert all(torch.equal(a, b) for a, b in zip(again, (dx, dwg, dwu)))


def test_glu_backward_f16_scale_follows_the_values(zkb):
    """zeros give zeros; an infinity stays in its token and does not set the scale; a captured call replayed on other values takes their scale"""
    n, e, f = 150, 72, 264
    x, wg, wu, gate, up, dh = glu_inputs(n, e, f, torch.float16, 8)
    x.mul_(64), wg.mul_(16), wu.mul_(16)
    outs = [torch.full_like(x, math.nan), torch.full_like(wg, math.nan), torch.full_like(wu, math.nan)]
    small = dh * 1e-5
    live = torch.zeros_like(dh)
    glu_back_call(zkb, 1, "silu", x, wg, wu, gate, up, live, *outs)
    assert all((o == 0).all() for o in outs)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        glu_back_call(zkb, 1, "silu", x, wg, wu, gate, up, live, *outs)
    for values in (small, dh, small):
        live.copy_(values)
        graph.replay()
        torch.cuda.synchronize()
        check_scaled("silu", x, wg, wu, gate, up, live, *outs)
    bad = small.clone()
    bad[7, 3], bad[9, 5] = math.inf, math.nan
    glu_back_call(zkb, 1, "silu", x, wg, wu, gate, up, bad, *outs)
    assert not outs[0][7].isfinite().any() and outs[0][9].isnan().all()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[[7, 9]] = False
    small[[7, 9]] = 0
    check_scaled("silu", x, wg, wu, gate, up, small, outs[0], None, None, keep)


# ---- the tail of the exact GELU ------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ("f16", "bf16"))
@pytest.mark.parametrize("n", (100, 300))
def test_gelu_far_below_zero(zkb, kind, n):
    """act(g) keeps its relative accuracy for gates from -8 to -3: the argument g / sqrt 2 is off by 2^-23 of itself, which moves erfc by g^2 = 64
    times that, and erfcf by 4 steps of 2^-23: below 2^-16 together.  In the derivative the fast exponential of -g^2 / 2 is off by 41 steps of
    2^-23 and its argument by 2^-23 of 32: below 2^-16 of each of its two terms."""
    code, t = TYPES[kind]
    f = 24
    g = torch.linspace(-8, -3, n, device="cuda").to(t)[:, None]
    one, zero = torch.ones(1, f, device="cuda", dtype=t), torch.zeros(1, f, device="cuda", dtype=t)
    up = torch.full((1, f), 16384.0, device="cuda", dtype=t)
    h, gate, u = (torch.empty(n, f, device="cuda", dtype=t) for _ in range(3))
    glu_call(zkb, code, "gelu", g, one, up / g.abs().max(), h, gate, u)
    assert torch.equal(gate, g.expand(n, f))
    G = g.double()
    cdf = 0.5 * torch.special.erfc(-G / math.sqrt(2))
    prod = G * cdf * (G @ (up / g.abs().max()).double())
    near(h, prod, t, 2.0 ** -16 * prod.abs())
    pdf = torch.exp(-0.5 * G * G) / math.sqrt(2 * math.pi)
    # one channel, so that dx is dg (weights 1 and 0) or du (0 and 1) itself
    dh, ones, dx = torch.full((n, 1), 256.0, device="cuda", dtype=t), torch.ones(n, 1, device="cuda", dtype=t), torch.empty(n, 1, device="cuda", dtype=t)
    glu_back_call(zkb, code, "gelu", ones, one[:, :1], zero[:, :1], g, ones, dh, dx, None, None)
    want, size = 256 * (cdf + G * pdf), 256 * (cdf + G.abs() * pdf)
    extra = 2.0 ** -39 * size.max() if kind == "f16" else 0.0
    near(dx, want, t, half_step(t) * want.abs() + 2.0 ** -15 * size + extra)
    glu_back_call(zkb, code, "gelu", ones, zero[:, :1], one[:, :1], g, ones, dh, dx, None, None)
    want = 256 * G * cdf
    near(dx, want, t, half_step(t) * want.abs() + 2.0 ** -16 * want.abs() + extra)


# ---- gates at the ends of the type ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind,far", (("bf16", 1e30), ("bf16", 1e20), ("bf16", 1e13), ("bf16", 200.0), ("f16", 60000.0), ("f16", 200.0)))
def test_glu_gates_far_from_zero(zkb, act, kind, far):
    """act is the identity or zero there and its derivative one or zero, whatever the powers of g do on the way (f16: within its range)"""
    code, t = TYPES[kind]
    n, f = 130, 16
    g = torch.full((n, 1), far, device="cuda").to(t)
    g[1::2] *= -1
    one, zero, ones = torch.ones(1, f, device="cuda", dtype=t), torch.zeros(1, f, device="cuda", dtype=t), torch.ones(n, 1, device="cuda", dtype=t)
    for rows in (slice(0, 2), slice(0, n)):
        x = g[rows]
        m = x.shape[0]
        h, gate, up = (torch.empty(m, f, device="cuda", dtype=t) for _ in range(3))
        glu_call(zkb, code, act, x, one, one, h, gate, up)
        assert torch.equal(gate, x.expand(m, f))
        if far * far < torch.finfo(t).max:
            assert torch.equal(h, (x.clamp(min=0) * x).expand(m, f))
        dx = torch.empty(m, 1, device="cuda", dtype=t)
        glu_back_call(zkb, code, act, ones[:m], one[:, :1], zero[:, :1], x, ones[:m], ones[:m], dx, None, None)
        assert torch.equal(dx, (x > 0).to(t))
        glu_back_call(zkb, code, act, ones[:m], zero[:, :1], one[:, :1], x, ones[:m], ones[:m], dx, None, None)
        assert torch.equal(dx, x.clamp(min=0))


# ---- calls beside one another ----------------------------------------------------------------------------------------------------------------------


def widths(z, t, code, cols, seed):
    r, y, pg, wg, gv, dz, dr = norm_inputs(40, cols, t, t, "channel", True, seed)
    outs = [torch.zeros_like(r), torch.zeros_like(r), torch.zeros_like(gv), torch.zeros_like(pg), torch.zeros_like(wg), torch.zeros_like(r), torch.zeros_like(r)]

    def go(st=None):
        norm_call(z, code, code, r, y, True, pg, "channel", gv, 0.7, wg, 1e-5, outs[5], outs[6], None, None, st=st)
        back_call(z, code, code, r, y, True, pg, "channel", gv, 0.7, wg, 1e-5, dz, dr, *outs[:5], st=st)
    return go, outs


def test_norms_of_different_widths_from_two_threads(zkb):
    """narrow and wide rows run the same kernel with rings of different sizes: neither call's launch depends on the other's"""
    made = [widths(zkb, torch.bfloat16, 2, cols, cols) for cols in (64, 2560)] + [widths(zkb, torch.float32, 0, cols, cols) for cols in (96, 2048)]
    for go, _ in made:
        go()
    torch.cuda.synchronize()
    want = [[o.clone() for o in outs] for _, outs in made]
    streams, errors = [torch.cuda.Stream() for _ in made], []

    def work(go, st):
        try:
            torch.cuda.set_device(0)
            for _ in range(400):
                go(st.cuda_stream)
            st.synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(go, st)) for (go, _), st in zip(made, streams)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for (_, outs), w in zip(made, want) for a, b in zip(outs, w))


def test_norms_of_different_widths_in_one_graph(zkb):
    made = [widths(zkb, torch.bfloat16, 2, cols, cols) for cols in (2560, 64, 2048, 128)]
    for go, _ in made:
        go()
    torch.cuda.synchronize()
    want = [[o.clone() for o in outs] for _, outs in made]
    for _, outs in made:
        for o in outs:
            o.zero_()
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        for go, _ in made:
            go()
    widths(zkb, torch.bfloat16, 2, 8, 1)[0]()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for (_, outs), w in zip(made, want) for a, b in zip(outs, w))


# ---- a call that failed ------------------------------------------------------------------------------------------------------------------------------


def test_a_call_that_failed_leaves_the_next_one_alone(zkb):
    """an allocation that cannot be met is that call's error, and not the next launch's"""
    q = torch.randn(1, 5, 2, 64, device="cuda")
    out, again, freq = torch.zeros_like(q), torch.zeros_like(q), rope_freq(64)
    rope_call(zkb, 0, [(q, out)], 1, 5, 64, 64, False, freq, 1.0, None, 0, 5, False)
    p = ctypes.c_void_p()
    with pytest.raises(zkb.ZkbError):
        zkb.call("zkb_malloc", ctypes.byref(p), ctypes.c_size_t(1 << 46))
    rope_call(zkb, 0, [(q, again)], 1, 5, 64, 64, False, freq, 1.0, None, 0, 5, False)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


# ---- waits that ran out -----------------------------------------------------------------------------------------------------------------------------------


def wait_word(zkb):
    """the word that kernels raise, in host memory"""
    where = getattr(zkb.lib(), "_ZN3zkb2tc9wait_flagEv")
    where.restype = ctypes.POINTER(ctypes.c_int)
    return where().contents


def test_a_wait_that_ran_out_is_told_to_everyone(zkb):
    """the word raised by the host, as a kernel would: each call and each wait of the library, on each thread, says so until it is reset; none runs"""
    z = zkb
    q = torch.randn(1, 5, 2, 64, device="cuda")
    out, freq = torch.full_like(q, 3.0), rope_freq(64)
    x, wg, wu, gate, up, dh = glu_inputs(9, 16, 24, torch.bfloat16, 1)
    h = torch.full((9, 24), 3.0, device="cuda", dtype=torch.bfloat16)
    r, y, pg, gg, gv, dz, dr = norm_inputs(4, 64, torch.float32, torch.float32, "none", True, 1)
    zed = torch.full_like(r, 3.0)
    host = torch.zeros(4)
    word = wait_word(z)
    assert z.call("zkb_wait_status", 0) == 0 and z.call("zkb_wait_status", 1) == 0
    calls = [lambda: rope_call(z, 0, [(q, out)], 1, 5, 64, 64, False, freq, 1.0, None, 0, 5, False),
             lambda: glu_call(z, 2, "silu", x, wg, wu, h, None, None),
             lambda: glu_back_call(z, 2, "silu", x, wg, wu, gate, up, dh, h, None, None),
             lambda: norm_call(z, 0, 0, r, None, False, None, "none", None, 1.0, None, 1e-5, None, zed, None, None),
             lambda: back_call(z, 0, 0, r, y, True, pg, "none", None, 1.0, gg, 1e-5, dz, dr, zed, None, None, None, None),
             lambda: z.call("zkb_sync", z._p(stream())),
             lambda: z.call("zkb_memcpy_d2h", z._p(host.data_ptr()), z._p(q.data_ptr()), z.sz(16), z._p(stream())),
             lambda: z.call("zkb_wait_status", 0)]
    told = []

    def everything():
        for c in calls:
            try:
                c()
                told.append("nothing")
            except z.ZkbError as e:
                told.append(e.code if "ran out" in e.msg else e.msg)
    word.value = 1
    try:
        everything()
        other = threading.Thread(target=everything)
        other.start()
        other.join()
        assert told == [z.ERR_CUDA] * 2 * len(calls), told
        torch.cuda.synchronize()
        assert all((v == 3).all() for v in (out, h, zed))
        with pytest.raises(z.ZkbError):
            z.call("zkb_wait_status", 1)
    finally:
        word.value = 0
    for c in calls:
        c()


def test_a_wait_that_nothing_ends(zkb, tmp_path):
    """a block waits on barriers that nobody arrives at, by one thread and by a warp: both waits end, the kernel does, and the library says so"""
    import os
    import shutil
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("needs nvcc")
    source = tmp_path / "wait.cu"
    source.write_text("""
#include "tensorcore.cuh"
#include <cstdio>
using namespace zkb;
__global__ void lonely(int* flag, int* ended, bool by_warp) {
    __shared__ uint64_t bar;
    __shared__ int dead;
    const uint32_t at = tc::smem_address(&bar);
    if (threadIdx.x == 0) {
        tc::barrier_init(at, 1);
        dead = 0;
    }
    __syncthreads();
    const tc::Watch watch = {&dead, flag};
    bool fine = true;
    if (by_warp) fine = tc::barrier_wait_warp(at, 0, watch);
    else if (threadIdx.x == 0) fine = tc::barrier_wait(at, 0, watch);
    if (threadIdx.x == 0) *ended = !fine && dead;
}
int main() {
    int* const flag = tc::wait_flag();
    int *ended, said[6], n = 0;
    if (!flag || cudaMalloc(&ended, 8) != cudaSuccess || cudaMemset(ended, 0, 8) != cudaSuccess) return 1;
    for (int w = 0; w < 2; ++w) {
        said[n++] = zkb_wait_status(0);
        lonely<<<1, 32>>>(flag, ended + w, w == 1);
        said[n++] = zkb_sync(nullptr);
        said[n++] = zkb_wait_status(1);
    }
    int got[2];
    if (zkb_memcpy_d2h(got, ended, 8, nullptr) != ZKB_OK) return 2;
    printf("%d %d | %d %d %d %d %d %d\\n", got[0], got[1], said[0], said[1], said[2], said[3], said[4], said[5]);
    return 0;
}
""")
    lib = root / "zkllm-ccs2024_b200" / "lib"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", str(root / "zkllm-ccs2024_b200" / "csrc"), str(source), "-o", str(tmp_path / "wait"),
                    "-L", str(lib), "-lzkllm_b200", "-Xlinker", f"-rpath={lib}"], check=True, timeout=300)
    res = subprocess.run([str(tmp_path / "wait")], capture_output=True, text=True, timeout=60)
    e = zkb.ERR_CUDA
    assert res.returncode == 0 and res.stdout.strip() == f"1 1 | 0 {e} {e} 0 {e} {e}", res.stdout + res.stderr


# ---- the side input of the rmsnorm stage ----------------------------------------------------------------------------------------------------------------


def test_rms_inv_refuses_what_its_file_cannot_hold(tmp_path):
    """a row of zeros with a tiny eps has an inverse beyond 32 bits: the stage ends with an error and writes nothing; at the border it is exact"""
    import subprocess

    import numpy as np
    from tests.test_gpu_drivers import BIN, save_int
    x = np.ones((4, 8), dtype=np.int64) * 65536
    x[2] = 0
    save_int(tmp_path / "x.bin", x)
    out = tmp_path / "rms_inv_temp.bin"
    for eps, fits in ((1e-10, False), (1e-30, False), (4e-9, True)):
        res = subprocess.run([str(BIN / "zkllm-driver"), "rms-inv", "x.bin", "4", "8", str(eps)], cwd=tmp_path, capture_output=True, text=True, timeout=120)
        assert (res.returncode == 0) == fits and out.exists() == fits, res.stderr
    got = np.fromfile(out, dtype=np.int32).astype(np.float64)
    want = 65536.0 / np.sqrt(((x / 65536.0) ** 2).mean(axis=1) + np.float64(np.float32(4e-9)))
    assert np.abs(got - want).max() <= 0.5 + 2.0 ** -20 * want.max()
