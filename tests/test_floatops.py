"""CPU: what the float operators (zkb_rope, zkb_block_norm, zkb_glu and their gradients) refuse before they touch the device, and the
host arithmetic of zkb_rope_frequencies."""
import ctypes
import math

import numpy as np
import pytest

P = 1 << 20          # an address that is never followed: every call here ends before its first access


def refused(zkb, code, name, *args):
    with pytest.raises(zkb.ZkbError) as e:
        zkb.call(name, *args)
    assert e.value.code == code, e.value.msg


def rope(zkb, dtype=2, tensors=None, n=1, batch=1, tokens=1, head_dim=8, rotary=8, freq=P):
    if tensors is None:
        tensors = zkb.rope_tensors((P, P, 1, (8, 8, 8), (8, 8, 8)))
    return ("zkb_rope", dtype, tensors, n, batch, tokens, head_dim, rotary, 0, freq, 1.0, None, 0, 0, 0, None)


def test_rope_refusals(zkb):
    z = zkb
    refused(z, z.ERR_ARG, *rope(z, dtype=3))
    refused(z, z.ERR_ARG, *rope(z, dtype=-1))
    refused(z, z.ERR_LIMIT, *rope(z, n=5))
    for rotary in (0, 3, 10):
        refused(z, z.ERR_DIM, *rope(z, rotary=rotary))
    refused(z, z.ERR_LIMIT, *rope(z, head_dim=8194, rotary=8194))
    refused(z, z.ERR_LIMIT, *rope(z, batch=1 << 16, tokens=1 << 16))
    refused(z, z.ERR_ARG, *rope(z, freq=None))
    assert z.call(*rope(z, tokens=0)) == 0 and z.call(*rope(z, batch=0)) == 0 and z.call(*rope(z, n=0)) == 0


def norm(dtype=2, gains=2, rows=2, cols=8, x=P, ldx=8, y=P, post=1, post_gain=P, kind=1, gate=P, ldg=8, scale=1.0, pre=1, pre_gain=P, eps=1e-5, z=P, post_inv=None):
    return ("zkb_block_norm", dtype, gains, rows, cols, x, ldx, y, 8, post, post_gain, kind, gate, ldg, scale, pre, pre_gain, eps, P, 8, z, 8, post_inv, None, None)


def test_block_norm_refusals(zkb):
    z = zkb
    for bad in (dict(dtype=7), dict(gains=1), dict(eps=0.0), dict(eps=math.nan), dict(eps=math.inf), dict(scale=math.inf), dict(kind=4), dict(kind=-1),
                dict(kind=0), dict(gate=None), dict(y=None), dict(post=0), dict(pre=0), dict(pre=0, pre_gain=None), dict(x=None),
                dict(y=None, post=0, post_gain=None), dict(post=0, post_gain=None, post_inv=P)):
        refused(z, z.ERR_ARG, *norm(**bad))
    refused(z, z.ERR_LIMIT, *norm(cols=16385))
    refused(z, z.ERR_LIMIT, *norm(rows=1 << 31))
    refused(z, z.ERR_DIM, *norm(ldx=7))
    assert z.call(*norm(rows=0)) == 0 and z.call(*norm(cols=0)) == 0


def norm_back(dtype=2, gains=2, rows=2, cols=8, r=P, y=P, post=1, post_gain=P, kind=1, gate=P, pre=1, pre_gain=P, eps=1e-5, dz=P, dr=P, dx=P, dy=P,
              dgate=P, dpost=P, dpre=P):
    return ("zkb_block_norm_backward", dtype, gains, rows, cols, r, 8, y, 8, post, post_gain, kind, gate, 8, 1.0, pre, pre_gain, eps, dz, 8, dr, 8, dx, 8, dy, 8,
            dgate, 8, dpost, dpre, None)


def test_block_norm_backward_refusals(zkb):
    z = zkb
    no_branch = dict(y=None, post=0, post_gain=None, kind=0, gate=None, dy=None, dgate=None, dpost=None)
    for bad in (dict(dtype=7), dict(gains=0, dtype=1, eps=-1.0), dict(pre=0), dict(pre=0, dz=None, pre_gain=None), {**no_branch, "dy": P},
                {**no_branch, "dgate": P}, {**no_branch, "dpost": P}, dict(kind=0, gate=None), dict(post=0, post_gain=None)):
        refused(z, z.ERR_ARG, *norm_back(**bad))
    refused(z, z.ERR_LIMIT, *norm_back(cols=20000))
    assert z.call(*norm_back(cols=0)) == 0


def glu(dtype=2, act=0, tokens=2, e=8, f=8, x=P, ldx=8, wg=P, h=P, gate=None, up=None):
    return ("zkb_glu", dtype, act, tokens, e, f, x, ldx, wg, 8, P, 8, h, 8, gate, 8, up, 8, None)


def test_glu_refusals(zkb):
    z = zkb
    for bad in (dict(dtype=0), dict(dtype=3), dict(act=4), dict(act=-1), dict(gate=P), dict(up=P), dict(x=None)):
        refused(z, z.ERR_ARG, *glu(**bad))
    refused(z, z.ERR_DIM, *glu(ldx=7))
    for big in (dict(tokens=(1 << 22) + 1), dict(e=(1 << 20) + 1), dict(f=(1 << 20) + 1)):
        refused(z, z.ERR_LIMIT, *glu(**big))
    assert z.call(*glu(tokens=0)) == 0 and z.call(*glu(f=0)) == 0

    def back(dtype=2, act=0, dwu=P, ldx=8, e=8):
        return ("zkb_glu_backward", dtype, act, 2, e, 8, P, ldx, P, 8, P, 8, P, 8, P, 8, P, 8, P, 8, P, 8, dwu, 8, None)
    for bad in (dict(dtype=0), dict(act=9), dict(dwu=None)):
        refused(z, z.ERR_ARG, *back(**bad))
    refused(z, z.ERR_DIM, *back(ldx=3))
    assert z.call(*back(e=0)) == 0


def frequencies(zkb, scaling, n, base=10000.0, factor=4.0, original=4096.0, fast=32.0, slow=1.0):
    f, m = np.zeros(n // 2), ctypes.c_float()
    zkb.call("zkb_rope_frequencies", scaling, n, base, factor, original, fast, slow, f.ctypes.data, ctypes.addressof(m))
    return f, m.value


def test_rope_frequencies(zkb):
    n = 128
    i = np.arange(n // 2)
    plain = 10000.0 ** (-2.0 * i / n)
    f, m = frequencies(zkb, 0, n)
    assert np.allclose(f, plain, rtol=1e-14, atol=0) and m == 1.0
    f, m = frequencies(zkb, 1, n)
    assert np.allclose(f, plain / 4, rtol=1e-14, atol=0) and m == 1.0
    f, m = frequencies(zkb, 2, n)
    assert np.allclose(f, (10000.0 * 4 ** (n / (n - 2))) ** (-2.0 * i / n), rtol=1e-13, atol=0)
    # the slowest pair is stretched by exactly the factor, the fastest not at all
    assert math.isclose(f[-1], plain[-1] / 4, rel_tol=1e-12) and f[0] == 1.0
    f, m = frequencies(zkb, 3, n)
    turns = 4096 * plain / (2 * math.pi)
    assert np.allclose(f[turns > 64], plain[turns > 64], rtol=1e-14, atol=0) and np.allclose(f[turns < 0.5], plain[turns < 0.5] / 4, rtol=1e-14, atol=0)
    assert np.all(np.diff(f) < 0) and np.all(f <= plain * (1 + 1e-15)) and np.all(f >= plain / 4 * (1 - 1e-15))
    assert math.isclose(m, 0.1 * math.log(4) + 1, rel_tol=1e-7)
    assert frequencies(zkb, 2, 2)[0][0] == 1.0 and frequencies(zkb, 3, 2)[0].size == 1


def test_rope_frequencies_refusals(zkb):
    z = zkb
    f, m = np.zeros(64), ctypes.c_float()
    good = [0, 8, 10000.0, 4.0, 4096.0, 32.0, 1.0, f.ctypes.data, ctypes.addressof(m)]
    for at, value, code in ((0, 4, z.ERR_ARG), (0, -1, z.ERR_ARG), (1, 0, z.ERR_DIM), (1, 7, z.ERR_DIM), (2, 1.0, z.ERR_ARG), (2, math.nan, z.ERR_ARG),
                            (7, None, z.ERR_ARG), (8, None, z.ERR_ARG)):
        refused(z, code, "zkb_rope_frequencies", *[value if i == at else v for i, v in enumerate(good)])
    for scaling, at, value in ((1, 3, 0.5), (2, 3, math.inf), (3, 4, 0.0), (3, 5, 1.0), (3, 6, 0.0), (3, 5, math.inf)):
        refused(z, z.ERR_ARG, "zkb_rope_frequencies", scaling, *[value if i == at else v for i, v in enumerate(good)][1:])
