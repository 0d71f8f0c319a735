"""Layers of token models without a GPU: refusals of the entry points and of the tensor functions, workspace sizes, and the
64-bit reference's backward formulas against differences of its forward formulas."""
import ctypes as C

import pytest
import tokens_ref as R
import torch

from cutagi_b200 import capi, ops
from cutagi_b200.capi import TagiError, lib

P = 4096          # an aligned address that is never read: every call below is refused on the host
f = C.c_float


def refused(name, *args):
    with pytest.raises(TagiError) as e:
        getattr(lib, name)(*args)
    assert e.value.code == 1
    return str(e.value)


def ln_args(**kw):
    a = dict(R=4, n=8, bias=1, eps=1e-5, p=[P] * 10)
    a.update(kw)
    return a["R"], a["n"], a["bias"], f(a["eps"]), *a["p"], None


def test_layer_norm_refusals():
    refused("tagi_ln_fwd", *ln_args(R=-1))
    refused("tagi_ln_fwd", *ln_args(n=1))
    refused("tagi_ln_fwd", *ln_args(eps=-1.0))
    refused("tagi_ln_fwd", *ln_args(eps=float("nan")))
    refused("tagi_ln_fwd", *ln_args(R=(1 << 30) + 1))
    refused("tagi_ln_fwd", *ln_args(n=(1 << 24) + 1))
    for i in range(10):
        for bad in (None, P + 2):
            refused("tagi_ln_fwd", *ln_args(p=[bad if j == i else P for j in range(10)]))


def test_layer_norm_backward_refusals():
    def args(R_=4, n=8, bias=1, su=1, p=None, ws=P, size=1 << 30):
        p = p or [P] * 15
        return (R_, n, bias, su, f(1e-5), *p, ws, size, None)
    refused("tagi_ln_bwd", *args(R_=-1))
    refused("tagi_ln_bwd", *args(n=1))
    refused("tagi_ln_bwd", *args(R_=2 ** 31 - 1))
    refused("tagi_ln_bwd", *args(n=2 ** 31 - 1))
    assert lib.tagi_ln_bwd_workspace_bytes(2 ** 31 - 1, 8) == lib.tagi_ln_bwd_workspace_bytes(8, 2 ** 31 - 1) == 0
    for i in range(15):
        if i != 4:      # the Jacobian may be NULL
            refused("tagi_ln_bwd", *args(p=[None if j == i else P for j in range(15)]))
        refused("tagi_ln_bwd", *args(p=[P + 1 if j == i else P for j in range(15)]))
    need = lib.tagi_ln_bwd_workspace_bytes(1000, 512)
    assert need > 0 and need % 16 == 0
    refused("tagi_ln_bwd", *args(R_=1000, n=512, ws=None))
    refused("tagi_ln_bwd", *args(R_=1000, n=512, ws=P + 4))
    refused("tagi_ln_bwd", *args(R_=1000, n=512, size=need - 1))
    assert lib.tagi_ln_bwd_workspace_bytes(1, 512) == 0 and lib.tagi_ln_bwd_workspace_bytes(0, 512) == 0


def test_route_refusals():
    def args(T=100, E=8, k=2, p=None, ws=P, size=1 << 30):
        return (T, E, k, *(p or [P] * 8), ws, size, None)
    for kw in (dict(T=-1), dict(E=0), dict(E=1025), dict(k=0), dict(k=9), dict(E=64, k=33), dict(T=1 << 30, k=4), dict(T=2 ** 31 - 1, k=1)):
        refused("tagi_route_fwd", *args(**kw))
    for i in range(8):
        if i != 1:      # the variances may be NULL
            refused("tagi_route_fwd", *args(p=[None if j == i else P for j in range(8)]))
        refused("tagi_route_fwd", *args(p=[P + 2 if j == i else P for j in range(8)]))
    need = lib.tagi_route_workspace_bytes(100, 8, 2)
    assert need > 0
    refused("tagi_route_fwd", *args(ws=None))
    refused("tagi_route_fwd", *args(size=need - 1))
    assert lib.tagi_route_workspace_bytes(1, 8, 2) == 0
    for kw in (dict(T=-1), dict(E=0), dict(k=9)):
        a = dict(T=4, E=8, k=2, **{}) | kw
        refused("tagi_route_bwd", a["T"], a["E"], a["k"], *[P] * 6, None)
    for i in range(6):
        refused("tagi_route_bwd", 4, 8, 2, *[None if j == i else P for j in range(6)], None)


def test_grouped_linear_refusals():
    def fwd(E=4, S=8, R_=8, K=16, N=16, bias=1, p=None, ws=P, size=1 << 30):
        return (E, S, R_, K, N, bias, *(p or [P] * 10), ws, size, None)
    for kw in (dict(E=0), dict(E=1025), dict(S=-1), dict(R_=-1), dict(K=0), dict(N=0), dict(K=(1 << 20) + 1),
               dict(S=(1 << 28) + 1), dict(R_=0)):
        refused("tagi_grouped_linear_fwd", *fwd(**kw))
    for i in range(10):
        if i != 1:      # the gather index may be NULL
            refused("tagi_grouped_linear_fwd", *fwd(p=[None if j == i else P for j in range(10)]))
        refused("tagi_grouped_linear_fwd", *fwd(p=[P + 2 if j == i else P for j in range(10)]))
    need = lib.tagi_grouped_linear_workspace_bytes(0, 4, 1000, 500, 64, 16)
    assert need >= 500 * 64 * 4 and lib.tagi_grouped_linear_workspace_bytes(0, 4, 0, 500, 64, 16) == 0
    assert lib.tagi_grouped_linear_workspace_bytes(0, 4, 1 << 30, 500, 64, 16) == lib.tagi_grouped_linear_workspace_bytes(3, 4, 8, 8, 64, 16) == 0
    for kw in (dict(ws=None), dict(ws=P + 4), dict(size=need - 1)):
        refused("tagi_grouped_linear_fwd", *fwd(S=1000, R_=500, K=64, **kw))
    refused("tagi_grouped_linear_fwd", *fwd(R_=7, p=[P, None] + [P] * 8))     # no gather index: R must equal S

    def state(E=4, S=8, K=16, N=16, p=None, ws=P, size=1 << 40):
        return (E, S, K, N, *(p or [P] * 7), ws, size, None)
    for kw in (dict(E=0), dict(S=-1), dict(K=0), dict(N=0)):
        refused("tagi_grouped_linear_bwd_state", *state(**kw))
    for i in range(7):
        if i != 2:
            refused("tagi_grouped_linear_bwd_state", *state(p=[None if j == i else P for j in range(7)]))
        refused("tagi_grouped_linear_bwd_state", *state(p=[P + 2 if j == i else P for j in range(7)]))

    def param(E=4, S=8, R_=8, K=16, N=16, bias=1, p=None, ws=P, size=1 << 40):
        return (E, S, R_, K, N, bias, *(p or [P] * 11), ws, size, None)
    for which, name, args in ((1, "tagi_grouped_linear_bwd_state", state), (2, "tagi_grouped_linear_bwd_param", lambda **kw: param(R_=1000, **kw))):
        need = lib.tagi_grouped_linear_workspace_bytes(which, 4, 1000, 1000, 16, 16)
        assert need > 0 and lib.tagi_grouped_linear_workspace_bytes(which, 4, 8, 8, 16, 16) == 0
        for kw in (dict(ws=None), dict(ws=P + 4), dict(size=need - 1)):
            refused(name, *args(S=1000, **kw))
    for kw in (dict(E=0), dict(S=-1), dict(K=0), dict(N=0), dict(R_=0)):
        refused("tagi_grouped_linear_bwd_param", *param(**kw))
    for i in range(11):
        if i != 1:
            refused("tagi_grouped_linear_bwd_param", *param(p=[None if j == i else P for j in range(11)]))
        refused("tagi_grouped_linear_bwd_param", *param(p=[P + 2 if j == i else P for j in range(11)]))


@pytest.mark.parametrize("name, ptrs, optional", [("tagi_combine_fwd", 7, ()), ("tagi_combine_bwd", 10, (3,)),
                                                  ("tagi_dispatch_bwd", 6, (1,))])
def test_combine_refusals(name, ptrs, optional):
    for T, k, N, S in ((-1, 2, 8, 8), (4, 0, 8, 8), (4, 2, 0, 8), (4, 2, 8, -1), (1 << 30, 4, 8, 8), (2 ** 31 - 1, 1, 8, 8),
                       (4, 2, 2 ** 31 - 1, 8)):
        refused(name, T, k, N, S, *[P] * ptrs, None)
    for i in range(ptrs):
        if i not in optional:
            refused(name, 4, 2, 8, 8, *[None if j == i else P for j in range(ptrs)], None)
        refused(name, 4, 2, 8, 8, *[P + 2 if j == i else P for j in range(ptrs)], None)


def test_tensor_functions_refuse_what_the_kernels_cannot_read():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):      # host tensors
        ops.layer_norm(z(8), z(8), z(8), z(8), z(4, 8), z(4, 8))
    with pytest.raises(ValueError, match="pair"):
        ops.layer_norm(z(8), z(8), z(8), None, z(4, 8), z(4, 8))
    with pytest.raises(ValueError, match="two dimensions"):
        ops.layer_norm(z(8), z(8), None, None, z(8), z(8))
    with pytest.raises(ValueError):
        ops.route(z(4, 8), z(4, 8), 2)
    with pytest.raises(ValueError):
        ops.grouped_linear(z(2, 8, 8), z(2, 8, 8), None, None, z(4, 8), z(4, 8), z(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.grouped_linear(z(8, 8), z(8, 8), None, None, z(4, 8), z(4, 8), z(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.combine(z(4, 2, dtype=torch.int32), z(4, 2), z(4, 2), z(8, 8), z(8, 8))


def test_tensor_functions_refuse_sizes_that_32_bits_do_not_hold():
    class Long:       # what the checks look at of a tensor that no test could allocate
        def __init__(self, *shape):
            self.shape = shape

        def dim(self):
            return len(self.shape)

        def get_device(self):
            return 0

        def numel(self):
            n = 1
            for s in self.shape:
                n *= s
            return n
    z, long = torch.zeros, 2 ** 32 + 4
    for call in (lambda: ops.layer_norm(z(8), z(8), None, None, Long(long, 8), None),
                 lambda: ops.route(Long(long, 8), None, 2),
                 lambda: ops.grouped_linear(Long(2, 8, 8), None, None, None, Long(long, 8), None, None),
                 lambda: ops.grouped_linear(Long(2, 8, 8), None, None, None, z(4, 8), None, None, Long(long)),
                 lambda: ops.grouped_linear_state(Long(2, 8, 8), None, Long(long, 8), None, None),
                 lambda: ops.grouped_linear_param(Long(2, 8, 8), None, z(4, 8), Long(long, 8), None, None),
                 lambda: ops.combine(Long(4, 2), None, None, Long(long, 8), None),
                 lambda: ops.dispatch_backward(Long(long, 1), None, Long(4, 8), None)):
        with pytest.raises(ValueError, match="2\\^31"):
            call()


def test_empty_calls_touch_nothing():
    assert lib.tagi_ln_fwd(*ln_args(R=0, p=[P] * 4 + [None] * 6)) == 0
    assert lib.tagi_grouped_linear_fwd(4, 0, 0, 16, 16, 1, P, None, P, P, P, P, None, None, None, None, None, 0, None) == 0
    assert lib.tagi_grouped_linear_bwd_state(4, 0, 16, 16, P, P, None, None, None, None, None, None, 0, None) == 0
    assert lib.tagi_combine_fwd(0, 2, 8, 0, *[None] * 8) == 0
    assert lib.tagi_combine_bwd(0, 2, 8, 0, *[None] * 11) == 0
    assert lib.tagi_dispatch_bwd(0, 2, 8, 0, *[None] * 7) == 0
    assert lib.tagi_route_bwd(0, 8, 2, *[None] * 7) == 0


# --------------------------------------------------------------------------- the reference's gradients, by differences

def _rnd(*shape, seed):
    return torch.randn(*shape, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))


def _close(a, b):
    assert abs(float(a) - float(b)) <= 1e-7 * (abs(float(a)) + abs(float(b)) + 1e-3)


def test_router_deltas_are_the_gates_gradient():
    T, E, k, h = 6, 9, 4, 1e-6
    s, dg, dirn = _rnd(T, E, seed=1), _rnd(T, k, seed=2), _rnd(T, E, seed=3)
    expert, (g, _), *_ = R.route_fwd(s, None, k)
    (dm, _), (dv, _) = R.route_bwd(expert, g, dg, torch.ones(T, k), E)
    up, down = R.route_fwd(s + h * dirn, None, k), R.route_fwd(s - h * dirn, None, k)
    assert torch.equal(up[0], expert) and torch.equal(down[0], expert)
    _close((dm * dirn).sum(), (dg * (up[1][0] - down[1][0])).sum() / (2 * h))
    # variance deltas: the squares of the same Jacobian's entries
    for t in range(T):
        for j in range(k):
            e = torch.zeros(T, E, dtype=torch.float64)
            e[t, expert[t, j]] = h
            col = (R.route_fwd(s + e, None, k)[1][0][t] - R.route_fwd(s - e, None, k)[1][0][t]) / (2 * h)
            _close(dv[t, expert[t, j]], (col * col).sum())


def test_expert_layer_deltas_are_the_gradients():
    T, E, k, K, N, h = 5, 3, 2, 4, 6, 1e-6
    s = _rnd(T, E, seed=1)
    _, (g, _), (vg, _), offsets, token, pos = R.route_fwd(s, None, k)
    w, b, a, dy = _rnd(E, N, K, seed=2), _rnd(E, N, seed=3), _rnd(T, K, seed=4), _rnd(T, N, seed=5)
    va, one = torch.zeros(T, K), torch.ones(T, N, dtype=torch.float64)

    def run(w, b, a, g):
        (x, _), _ = R.grouped_fwd(w, w * 0, b, b * 0, a, va, offsets, token)
        return R.combine_fwd(pos, g, vg, x, x * 0)[0][0], x
    y, x = run(w, b, a, g)
    (dx, _), (dvx, _), (dg, _), _ = R.combine_bwd(pos, g, x, None, dy, one)
    (dr, _), (dvr, _) = R.grouped_state(w, None, dx, dvx, offsets)
    (da, _), _ = R.dispatch_bwd(pos, None, dr, dvr)
    (dw, _), _, (db, _), _ = R.grouped_param(torch.ones_like(w), torch.ones_like(b), a, dx, dvx, offsets, token)
    for i, (t, grad) in enumerate(((w, dw), (b, db), (a, da), (g, dg))):
        dirn = _rnd(*t.shape, seed=10 + i)
        args = [w, b, a, g]
        up, down = list(args), list(args)
        up[i], down[i] = t + h * dirn, t - h * dirn
        _close((grad * dirn).sum(), (dy * (run(*up)[0] - run(*down)[0])).sum() / (2 * h))


def test_layer_norm_deltas_are_the_gradients_at_fixed_statistics():
    n, rows, h, eps = 7, 4, 1e-6, 1e-3
    w, vw, b, vb = _rnd(n, seed=1), _rnd(n, seed=2).square(), _rnd(n, seed=3), _rnd(n, seed=4).square()
    a, va, dm = _rnd(rows, n, seed=5), _rnd(rows, n, seed=6).square(), _rnd(rows, n, seed=7)
    (z, _), (vz, _), (m, _), (v, _) = R.ln_fwd(w, vw, b, vb, a, va, eps)
    assert torch.allclose(m, a.mean(1)) and torch.allclose(v, a.var(1) + va.sum(1) / (n - 1))
    dmu, dvar, dw, dvw, db, dvb = [p[0] for p in R.ln_bwd(w, vw, vb, a, None, m, v, dm, -dm.square(), eps)]

    def run(w, b, a):
        return (a - m[:, None]) * (v[:, None] + eps).rsqrt() * w + b
    assert torch.allclose(run(w, b, a), z)
    for i, (t, grad) in enumerate(((w, dw / vw), (b, db / vb), (a, dmu))):
        dirn = _rnd(*t.shape, seed=20 + i)
        up, down = [w, b, a], [w, b, a]
        up[i], down[i] = t + h * dirn, t - h * dirn
        _close((grad * dirn).sum(), (dm * (run(*up) - run(*down))).sum() / (2 * h))
    # every output entry depends on one entry of each, so the variance deltas are the squares of the same factors
    assert torch.allclose(dvar, -dmu.square())


def test_capi_knows_the_sizes():
    assert capi.load().tagi_route_workspace_bytes(1 << 20, 1024, 8) < 1 << 20
    assert capi.load().tagi_ln_bwd_workspace_bytes(1 << 20, 4096) < 1 << 26
