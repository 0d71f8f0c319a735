"""Layers of token models on the GPU against the 64-bit formulas of tokens_ref (tolerances: its docstring), through the C ABI
with guard bands around every output, and as a whole expert layer."""
import ctypes as C

import pytest
import tokens_ref as R
import torch

pytestmark = pytest.mark.gpu
f32, i32 = torch.float32, torch.int32
EPS = 1e-5
SENT = -777.25


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cutagi_b200.capi import lib
    return lib


@pytest.fixture(autouse=True)
def no_wait_ran_out(lib):
    """The tensor-core kernels give a wait up after a second and leave a word about it: none may have."""
    from cutagi_b200 import capi
    yield
    assert capi.tc_status() == 0


class Guard:
    """An output with sentinels around it (and in it, until it is written)."""

    def __init__(self, *shape, dtype=f32, misalign=0):
        self.n, self.shape = 1, shape
        for s in shape:
            self.n *= s
        self.off = 64 + misalign
        self.sent = SENT if dtype == f32 else -777
        self.buf = torch.full((self.n + 128 + misalign,), self.sent, dtype=dtype, device="cuda")

    def ptr(self):
        return self.buf[self.off:].data_ptr()

    def get(self, whole=True):
        assert bool((self.buf[:self.off] == self.sent).all()) and bool((self.buf[self.off + self.n:] == self.sent).all()), \
            "guard band overwritten"
        out = self.buf[self.off:self.off + self.n].reshape(self.shape)
        assert not whole or not bool((out == self.sent).any()), "output not fully written"
        return out


class Gen:
    def __init__(self, seed, misalign=0):
        self.g, self.mis = torch.Generator(device="cuda").manual_seed(seed), misalign

    def _at(self, t):
        if not self.mis:
            return t
        b = torch.empty(t.numel() + self.mis, dtype=t.dtype, device="cuda")
        b[self.mis:] = t.reshape(-1)
        return b[self.mis:].reshape(t.shape)

    def n(self, *shape, scale=1.0, mean=0.0):
        return self._at(torch.randn(*shape, device="cuda", generator=self.g) * scale + mean)

    def u(self, *shape, lo=0.0, hi=1.0):
        return self._at(torch.rand(*shape, device="cuda", generator=self.g) * (hi - lo) + lo)


def p(t):
    return None if t is None else t.data_ptr()


def st():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------------------------------------------------ LayerNorm

def ln_params(g, n, bias):
    w = [g.n(n, scale=0.3, mean=1.0), g.u(n, lo=0.01, hi=0.3)]
    return w + ([g.n(n, scale=0.2), g.u(n, lo=0.01, hi=0.3)] if bias else [None, None])


# the borders of the kernels' row lengths (32, 64 ... 1024 threads with 16 entries each, and beyond), odd lengths, one row
LN_SIZES = [(1, 2), (3, 5), (9, 33), (7, 512), (7, 513), (5, 1024), (5, 1028), (3, 2047), (3, 2048), (2, 2052), (2, 4096),
            (3, 4097), (2, 8192), (2, 8196), (1, 16384), (2, 16385), (2, 20000), (1000, 64), (333, 768)]


@pytest.mark.parametrize("rows, n", LN_SIZES)
@pytest.mark.parametrize("bias, misalign", [(True, 0), (False, 0), (True, 1)])
def test_layer_norm_forward(lib, rows, n, bias, misalign):
    g = Gen(n + rows, misalign)
    mw, vw, mb, vb = ln_params(g, n, bias)
    ma, va = g.n(rows, n, scale=2.0, mean=0.7), g.u(rows, n, lo=0.01, hi=0.5)
    z, vz = Guard(rows, n, misalign=misalign), Guard(rows, n, misalign=misalign)
    m, v = Guard(rows), Guard(rows)
    lib.tagi_ln_fwd(rows, n, int(bias), C.c_float(EPS), p(mw), p(vw), p(mb), p(vb), p(ma), p(va), m.ptr(), v.ptr(), z.ptr(),
                    vz.ptr(), st())
    ref = R.ln_fwd(mw, vw, mb, vb, ma, va, C.c_float(EPS).value)
    for name, got, pair in zip(("mu_z", "var_z", "mu_row", "var_row"), (z, vz, m, v), ref):
        R.check(name, got.get(), pair, R.U)


def with_workspace(lib, name, which, E, S, rows, K, N, *args):
    """A pass of the grouped Linear layers with a guarded workspace full of NaN."""
    size = lib.tagi_grouped_linear_workspace_bytes(which, E, S, rows, K, N)
    ws = torch.full((size // 4 + 32,), torch.nan, device="cuda")
    ws[size // 4:] = SENT
    getattr(lib, name)(*args, p(ws), size, st())
    assert bool((ws[size // 4:] == SENT).all())


def grouped_fwd(lib, E, S, rows, K, N, *args):
    with_workspace(lib, "tagi_grouped_linear_fwd", 0, E, S, rows, K, N, E, S, rows, K, N, *args)


def grouped_state(lib, E, S, K, N, *args):
    with_workspace(lib, "tagi_grouped_linear_bwd_state", 1, E, S, S, K, N, E, S, K, N, *args)


def grouped_param(lib, E, S, rows, K, N, *args):
    with_workspace(lib, "tagi_grouped_linear_bwd_param", 2, E, S, rows, K, N, E, S, rows, K, N, *args)


def test_layer_norm_forward_of_a_constant_row(lib):
    """No spread at all: the variance is what the inputs' own variances give, zero with them at zero."""
    n = 256
    one, zero = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    ma, va = torch.full((2, n), 3.0, device="cuda"), torch.zeros(2, n, device="cuda")
    va[1] = 0.5
    z, vz, m, v = Guard(2, n), Guard(2, n), Guard(2), Guard(2)
    lib.tagi_ln_fwd(2, n, 0, C.c_float(EPS), p(one), p(zero), None, None, p(ma), p(va), m.ptr(), v.ptr(), z.ptr(), vz.ptr(), st())
    assert bool((z.get() == 0).all()) and bool((m.get() == 3).all()) and v.get()[0].item() == 0.0
    assert abs(v.get()[1].item() - 0.5 * n / (n - 1)) <= 16 * R.U


# chunks of rows: below, at and above the border of one chunk, many chunks
@pytest.mark.parametrize("rows, n", [(1, 2), (1, 4096), (15, 64), (16, 64), (17, 64), (33, 100), (257, 513), (5000, 36),
                                     (3000, 1001), (40, 20000)])
@pytest.mark.parametrize("bias, jcb, state, misalign", [(True, True, True, 0), (False, False, True, 0), (True, False, False, 0),
                                                        (True, True, True, 1)])
def test_layer_norm_backward(lib, rows, n, bias, jcb, state, misalign):
    g = Gen(7 * n + rows, misalign)
    mw, vw, _, vb = ln_params(g, n, bias)
    ma, j = g.n(rows, n, scale=2.0, mean=0.7), (g.u(rows, n) if jcb else None)
    m, v = ma.mean(1).contiguous(), g.u(rows, lo=0.5, hi=4.0)
    dm, dv = g.n(rows, n, scale=0.1), g.u(rows, n, lo=-0.1, hi=0.0)
    o = [Guard(rows, n, misalign=misalign) for _ in range(2)] + [Guard(n) for _ in range(4)]
    size = lib.tagi_ln_bwd_workspace_bytes(rows, n)
    ws = torch.full((size // 4 + 32,), SENT, device="cuda")
    lib.tagi_ln_bwd(rows, n, int(bias), int(state), C.c_float(EPS), p(mw), p(vw), p(vb), p(ma), p(j), p(m), p(v), p(dm), p(dv),
                    o[0].ptr() if state else None, o[1].ptr() if state else None, *[x.ptr() for x in o[2:]], p(ws), size, st())
    ref = R.ln_bwd(mw, vw, vb, ma, j, m, v, dm, dv, C.c_float(EPS).value)
    assert bool((ws[size // 4:] == SENT).all())
    for i, name in enumerate(("dmu", "dvar", "dmu_w", "dvar_w", "dmu_b", "dvar_b")):
        if (i < 2 and not state) or (i >= 4 and not bias):
            assert bool((o[i].get(whole=False) == SENT).all()), name
        else:
            R.check(name, o[i].get(), ref[i], R.sum_tol(rows if i >= 2 else 1))


def test_layer_norm_backward_without_rows_gives_zero_deltas(lib):
    n = 100
    w, o = torch.ones(n, device="cuda"), [Guard(n) for _ in range(4)]
    lib.tagi_ln_bwd(0, n, 1, 1, C.c_float(EPS), p(w), p(w), p(w), None, None, None, None, None, None, None, None,
                    *[x.ptr() for x in o], None, 0, st())
    assert all(bool((x.get() == 0).all()) for x in o)


# -------------------------------------------------------------------------------------------------------------- routing

def run_route(lib, ms, vs, k):
    T, E = ms.shape
    ints = [Guard(T, k, dtype=i32), Guard(E + 1, dtype=i32), Guard(T * k, dtype=i32), Guard(T, k, dtype=i32)]
    gates = [Guard(T, k), Guard(T, k)]
    size = lib.tagi_route_workspace_bytes(T, E, k)
    ws = torch.full((size // 4 + 32,), -777, dtype=i32, device="cuda")
    lib.tagi_route_fwd(T, E, k, p(ms), p(vs), ints[0].ptr(), gates[0].ptr(), gates[1].ptr(), ints[1].ptr(), ints[2].ptr(),
                       ints[3].ptr(), p(ws), size, st())
    assert bool((ws[size // 4:] == -777).all())
    return ints[0].get(), gates[0].get(), gates[1].get(), ints[1].get(), ints[2].get(), ints[3].get()


def check_route(lib, ms, vs, k):
    expert, g, vg, offsets, token, pos = run_route(lib, ms, vs, k)
    ref = R.route_fwd(ms, vs, k)
    for name, got, want in (("expert", expert, ref[0]), ("offsets", offsets, ref[3]), ("token", token, ref[4]), ("pos", pos, ref[5])):
        assert torch.equal(got.long(), want), name
    R.check("mu_g", g, ref[1], R.U)
    R.check("var_g", vg, ref[2], R.U)
    gen = Gen(3)
    dg, dvg = gen.n(*g.shape), gen.u(*g.shape, lo=-1.0, hi=0.0)
    none = expert < 0
    dg[none], dvg[none] = torch.nan, torch.inf       # deltas of slots without an expert have no part in anything
    dm, dv = Guard(*ms.shape), Guard(*ms.shape)
    T, E = ms.shape
    lib.tagi_route_bwd(T, E, k, p(expert), p(g), p(dg), p(dvg), dm.ptr(), dv.ptr(), st())
    want = R.route_bwd(expert, g, dg, dvg, E)
    R.check("dmu_s", dm.get(), want[0], (16 + 2 * k) * R.U)
    R.check("dvar_s", dv.get(), want[1], (16 + 4 * k) * R.U)


@pytest.mark.parametrize("T", [1, 31, 32, 33, 300, 5001])
@pytest.mark.parametrize("E, k", [(1, 1), (2, 2), (8, 2), (32, 4), (33, 1), (128, 8), (129, 5), (512, 3), (513, 2), (1000, 32), (1024, 1),
                                  (64, 8), (60, 16), (100, 9), (250, 12), (128, 17), (256, 20), (400, 8)])
def test_route(lib, T, E, k):
    g = Gen(T * 1000 + E)
    check_route(lib, g.n(T, E, scale=2.0), g.u(T, E), k)


def test_route_of_unaligned_scores(lib):
    g = Gen(8, misalign=1)
    check_route(lib, g.n(500, 64), g.u(500, 64), 4)


@pytest.mark.parametrize("E, k", [(16, 3), (128, 8), (130, 12), (64, 20), (600, 5)])
def test_route_ties(lib, E, k):
    g = Gen(E)
    check_route(lib, torch.round(g.n(301, E)), g.u(301, E), k)


@pytest.mark.parametrize("T", [20, 700])
def test_route_ties_and_barred_experts(lib, T):
    g = Gen(T)
    ms, vs = torch.round(g.n(T, 40)), g.u(T, 40)               # many equal scores, both zeros among them
    ms[::3] *= -1.0
    ms[1], ms[2], ms[3] = -torch.inf, torch.nan, torch.finfo(f32).min
    ms[4, :39], ms[5, ::2] = -torch.inf, torch.nan
    ms[6, 5] = torch.inf
    ms[7, [3, 9, 30]] = torch.inf
    ms[8:12] = torch.where(g.u(4, 40) < 0.9, -torch.inf, ms[8:12])
    check_route(lib, ms, vs, 6)
    check_route(lib, ms, None, 6)


def test_route_of_no_tokens(lib):
    offsets = Guard(9, dtype=i32)
    lib.tagi_route_fwd(0, 8, 2, None, None, None, None, None, offsets.ptr(), None, None, None, 0, st())
    assert bool((offsets.get() == 0).all())


def test_route_all_tokens_to_one_expert(lib):
    ms = torch.zeros(2000, 64, device="cuda")
    ms[:, 17] = 5.0
    check_route(lib, ms, None, 1)


# ------------------------------------------------------------------------------------------------------- grouped Linear

def spread(counts, lead=0, tail=0):
    """offsets of the given row counts, `lead` rows before the first and `tail` behind the last, and S."""
    o = torch.tensor([0] + counts).cumsum(0) + lead
    return o.to(i32).cuda(), int(o[-1]) + tail


# (rows of each expert, K, N): empty experts, single rows, tiles' borders, odd sizes, one feature, long contractions
GROUPED = [([1], 1, 1), ([1], 64, 32), ([2, 0, 1], 17, 33), ([0, 0, 5], 64, 64), ([3, 4, 8, 9], 128, 96), ([16, 17, 15, 0], 96, 130),
           ([0], 32, 32), ([64, 1, 63], 256, 128), ([40, 100, 7], 257, 65), ([128, 129, 127], 160, 256), ([300, 0, 5, 200], 100, 300),
           ([700], 64, 520), ([31, 257, 90], 1000, 72), ([5, 2], 4096, 64), ([256, 600], 512, 384), ([1000, 3], 33, 31)]


def guard_rows(out, r0, r1):
    """Rows r0 .. r1 - 1, after checking that the others are as they were."""
    t = out.get(whole=False)
    assert bool((t[:r0] == SENT).all()) and bool((t[r1:] == SENT).all()), "a row that no expert owns was written"
    assert not bool((t[r0:r1] == SENT).any())
    return t[r0:r1]


def sub(pair, r0, r1):
    return pair[0][r0:r1], pair[1][r0:r1]


@pytest.mark.parametrize("counts, K, N", GROUPED)
@pytest.mark.parametrize("bias, gather, misalign, lead, tail", [(True, True, 0, 0, 0), (False, False, 0, 2, 3), (True, True, 1, 0, 5)])
def test_grouped_linear(lib, counts, K, N, bias, gather, misalign, lead, tail):
    g = Gen(K * 31 + N, misalign)
    E = len(counts)
    offsets, S = spread(counts, lead, tail)
    r0, r1 = lead, S - tail
    rows = max(1, S // 2) if gather else S
    token = torch.randint(0, rows, (S,), device="cuda", generator=g.g).to(i32) if gather else None
    s = K ** -0.5
    mw, vw = g.n(E, N, K, scale=s), g.u(E, N, K, lo=0.1 * s * s, hi=s * s)
    mb, vb = (g.n(E, N, scale=0.1), g.u(E, N, lo=0.001, hi=0.1)) if bias else (None, None)
    ma, va = g.n(rows, K), g.u(rows, K, lo=0.001, hi=0.2)
    z, vz = Guard(S, N, misalign=misalign), Guard(S, N, misalign=misalign)
    grouped_fwd(lib, E, S, rows, K, N, int(bias), p(offsets), p(token), p(mw), p(vw), p(mb), p(vb), p(ma), p(va),
                                z.ptr(), vz.ptr())
    ref = R.grouped_fwd(mw, vw, mb, vb, ma, va, offsets, token)
    R.check("mu_z", guard_rows(z, r0, r1), sub(ref[0], r0, r1), R.sum_tol(K))
    R.check("var_z", guard_rows(vz, r0, r1), sub(ref[1], r0, r1), R.sum_tol(2 * K))

    dm, dv, jcb = g.n(S, N, scale=0.1), g.u(S, N, lo=-0.2, hi=0.0), (g.u(S, K) if bias else None)
    da, dva = Guard(S, K, misalign=misalign), Guard(S, K, misalign=misalign)
    grouped_state(lib, E, S, K, N, p(offsets), p(mw), p(jcb), p(dm), p(dv), da.ptr(), dva.ptr())
    ref = R.grouped_state(mw, jcb, dm, dv, offsets)
    R.check("dmu_a", guard_rows(da, r0, r1), sub(ref[0], r0, r1), R.sum_tol(N))
    R.check("dvar_a", guard_rows(dva, r0, r1), sub(ref[1], r0, r1), R.sum_tol(N))

    o = [Guard(E, N, K, misalign=misalign) for _ in range(2)] + [Guard(E, N) for _ in range(2)]
    grouped_param(lib, E, S, rows, K, N, int(bias), p(offsets), p(token), p(vw), p(vb), p(ma), p(dm), p(dv),
                                      *[x.ptr() for x in o])
    ref = R.grouped_param(vw, vb, ma, dm, dv, offsets, token)
    for i, name in enumerate(("dmu_w", "dvar_w", "dmu_b", "dvar_b")):
        if i < 2 or bias:
            R.check(name, o[i].get(), ref[i], R.sum_tol(max(counts)))
        else:
            assert bool((o[i].get(whole=False) == SENT).all())


@pytest.mark.parametrize("counts", [[1, 3], [20, 9], [70, 130]])
@pytest.mark.parametrize("K, N", [(37, 70), (64, 64)])
def test_grouped_linear_of_tensors_aligned_differently(lib, counts, K, N):
    """Each tensor begins at its own distance from a multiple of 16 bytes, behind a NaN."""
    from cutagi_b200 import ops

    def at(t, off):
        b = torch.full((t.numel() + 8,), torch.nan, device="cuda")
        b[off:off + t.numel()] = t.reshape(-1)
        return b[off:off + t.numel()].reshape(t.shape)
    g, E = Gen(K), len(counts)
    offsets, S = spread(counts)
    for d in range(4):
        mw, vw, a, va = at(g.n(E, N, K), 1 + d), at(g.u(E, N, K), 1 + (d + 1) % 4), at(g.n(S, K), 1 + (d + 2) % 4), at(g.u(S, K), 2)
        dm, dv = at(g.n(S, N), 1 + (d + 3) % 4), at(g.u(S, N), 3)
        got = (*ops.grouped_linear(mw, vw, None, None, a, va, offsets), *ops.grouped_linear_state(mw, None, dm, dv, offsets),
               *ops.grouped_linear_param(vw, None, a, dm, dv, offsets)[:2])
        ref = (*R.grouped_fwd(mw, vw, None, None, a, va, offsets, None), *R.grouped_state(mw, None, dm, dv, offsets),
               *R.grouped_param(vw, None, a, dm, dv, offsets, None))
        for x, pair, L in zip(got, ref, (K, 2 * K, N, N, max(counts), max(counts))):
            R.check(f"offset {d}", x, pair, R.sum_tol(L))


# experts on both sides of every border between the kernels (8, 14 and 48 rows) and of the widest tile (256), with rows that
# are aligned to 16 bytes in both, one or none of the two directions
@pytest.mark.parametrize("counts", [[8, 9, 14, 15, 48, 49, 0, 16, 17], [255, 256, 257, 512, 513, 3], [64, 65, 96, 33, 32, 31]])
@pytest.mark.parametrize("K, N", [(260, 132), (130, 67), (516, 1031), (129, 300)])
@pytest.mark.parametrize("bias, gather, misalign, lead, tail", [(True, True, 0, 1, 2), (True, False, 0, 0, 0)])
def test_grouped_linear_at_the_kernels_borders(lib, counts, K, N, bias, gather, misalign, lead, tail):
    test_grouped_linear(lib, counts, K, N, bias, gather, misalign, lead, tail)


@pytest.mark.parametrize("few, some", [(1, 64), (9, 30), (0, 70)])
def test_grouped_linear_of_1024_experts(lib, few, some):
    counts = [few] * 1024
    for e in (0, 31, 32, 500, 1023):
        counts[e] = some
    test_grouped_linear(lib, counts, 68, 40, True, True, 0, 0, 3)


def test_grouped_linear_of_many_tiles(lib):
    """More tiles than CTA pairs, so that each takes several in a row: of both kinds, many widths, all the experts' biases."""
    test_grouped_linear(lib, [1500, 0, 333, 2100, 7, 30, 900], 1100, 1030, True, True, 0, 0, 0)
    test_grouped_linear(lib, [40] * 30, 700, 2060, True, False, 0, 0, 0)


@pytest.mark.parametrize("counts, K, N", [([300], 3000, 100), ([60, 50], 100, 3000), ([5000, 30, 800], 24, 40), ([520, 0, 70], 1536, 1403),
                                          ([100] * 11, 2050, 513), ([49], 4100, 16), ([2000], 16, 300), ([9], 4100, 20), ([30, 0, 48], 2047, 300),
                                          ([20, 5, 40, 130], 1300, 1290)])
@pytest.mark.parametrize("bias, gather", [(True, True), (False, False)])
def test_grouped_linear_of_few_tiles_and_long_contractions(lib, counts, K, N, bias, gather):
    """Tiles that are cut along the contraction, because whole ones would leave most of the GPU idle."""
    test_grouped_linear(lib, counts, K, N, bias, gather, 0, 1, 1)


def big(*shape):
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GB of device memory")
    return torch.zeros(*shape, device="cuda")


@pytest.mark.parametrize("K, N", [(64, 4096), (4096, 64)])
def test_grouped_linear_row_offsets_past_32_bits(lib, K, N):
    g, counts = Gen(K), [7, 40, 250]
    S = 2 ** 19 + 300
    offsets, S = spread(counts, S - sum(counts))
    r0 = S - sum(counts)
    s = K ** -0.5
    mw, vw, vb = g.n(3, N, K, scale=s), g.u(3, N, K, hi=s * s), g.u(3, N)
    a, va, dm, dv = (big(S, n) for n in (K, K, N, N))
    for t in (a, va, dm, dv):
        t[r0:] = g.u(S - r0, t.shape[1])
    from cutagi_b200 import ops
    live = (offsets - r0).to(i32)
    z, vz = ops.grouped_linear(mw, vw, None, None, a, va, offsets)
    ref = R.grouped_fwd(mw, vw, None, None, a[r0:], va[r0:], live, None)
    R.check("mu_z", z[r0:], ref[0], R.sum_tol(K))
    R.check("var_z", vz[r0:], ref[1], R.sum_tol(2 * K))
    del z, vz, va
    da, dva = ops.grouped_linear_state(mw, None, dm, dv, offsets)
    ref = R.grouped_state(mw, None, dm[r0:], dv[r0:], live)
    R.check("dmu_a", da[r0:], ref[0], R.sum_tol(N))
    R.check("dvar_a", dva[r0:], ref[1], R.sum_tol(N))
    del da, dva
    got = ops.grouped_linear_param(vw, vb, a, dm, dv, offsets)
    for name, x, pair in zip(("dmu_w", "dvar_w", "dmu_b", "dvar_b"), got, R.grouped_param(vw, vb, a[r0:], dm[r0:], dv[r0:], live, None)):
        R.check(name, x, pair, R.sum_tol(max(counts)))
    del a, dm, dv
    torch.cuda.empty_cache()


def test_grouped_linear_weight_offsets_past_32_bits(lib):
    from cutagi_b200 import ops
    E, K, N = 516, 2048, 2048
    g, counts = Gen(2), [0] * (E - 3) + [5, 40, 60]
    offsets, S = spread(counts)
    mw, vw = big(E, N, K), big(E, N, K)
    s = K ** -0.5
    mw[-3:], vw[-3:] = g.n(3, N, K, scale=s), g.u(3, N, K, hi=s * s)
    a, va, dm, dv = g.n(S, K), g.u(S, K), g.n(S, N), g.u(S, N)
    z, vz = ops.grouped_linear(mw, vw, None, None, a, va, offsets)
    da, dva = ops.grouped_linear_state(mw, None, dm, dv, offsets)
    last = offsets[-4:]
    ref = (*R.grouped_fwd(mw[-3:], vw[-3:], None, None, a, va, last, None), *R.grouped_state(mw[-3:], None, dm, dv, last))
    for name, x, pair, L in zip(("mu_z", "var_z", "dmu_a", "dvar_a"), (z, vz, da, dva), ref, (K, 2 * K, N, N)):
        R.check(name, x, pair, R.sum_tol(L))
    del mw
    got = ops.grouped_linear_param(vw, None, a, dm, dv, offsets)
    for name, x, pair in zip(("dmu_w", "dvar_w"), got, R.grouped_param(vw[-3:], None, a, dm, dv, last, None)):
        R.check(name, x[-3:], pair, R.sum_tol(max(counts)))
        assert not bool(x[:-3].any())
    del got, vw
    torch.cuda.empty_cache()


def test_row_offsets_past_32_bits(lib):
    """LayerNorm and the combination with rows that begin behind 2^31 floats."""
    from cutagi_b200 import ops
    g, n, live = Gen(4), 4096, 40
    rows = 2 ** 19 + live
    a, va = big(rows, n), big(rows, n)
    a[-live:], va[-live:] = g.n(live, n), g.u(live, n)
    mw, vw, mb, vb = ln_params(g, n, True)
    z, vz, m, v = ops.layer_norm(mw, vw, mb, vb, a, va, EPS)
    for name, x, pair in zip(("mu_z", "var_z", "mu_row", "var_row"), (z, vz, m, v), R.ln_fwd(mw, vw, mb, vb, a[-live:], va[-live:], C.c_float(EPS).value)):
        R.check(name, x[-live:], pair, R.U)
    z.zero_(), vz.zero_()
    z[-live:], vz[-live:] = g.n(live, n), g.u(live, n)
    got = ops.layer_norm_backward(mw, vw, vb, a, None, m, v, z, vz, EPS)
    ref = R.ln_bwd(mw, vw, vb, a[-live:], None, m[-live:], v[-live:], z[-live:], vz[-live:], C.c_float(EPS).value)
    for i, name in enumerate(("dmu", "dvar", "dmu_w", "dvar_w", "dmu_b", "dvar_b")):   # the other rows' deltas are zero
        R.check(name, got[i][-live:] if i < 2 else got[i], ref[i], R.sum_tol(live if i >= 2 else 1))
    del got, z, vz
    torch.cuda.empty_cache()
    pos = torch.tensor([[rows - 1, 3], [rows - 2, rows - 30]], dtype=i32, device="cuda")
    mg, vg, dm, dv = g.u(2, 2), g.u(2, 2), g.n(2, n), g.u(2, n)
    few = torch.where(pos >= live, pos - (rows - live), -1)
    y = ops.combine(pos, mg, vg, a, va)
    for x, pair in zip(y, R.combine_fwd(few, mg, vg, a[-live:], va[-live:])):
        R.check("combine", x, pair, 12 * R.U)
    d = ops.dispatch_backward(pos, None, a, va)
    for x, pair in zip(d, R.dispatch_bwd(few, None, a[-live:], va[-live:])):
        R.check("dispatch", x, pair, 12 * R.U)
    got = ops.combine_backward(pos, mg, a, None, dm, dv)
    ref = R.combine_bwd(few, mg, a[-live:], None, dm, dv)
    for x, (want, M) in zip(got[:2], ref[:2]):
        named = ~torch.isnan(want[:, 0])
        R.check("rows", x[-live:][named], (want[named], M[named]), 8 * R.U)
    for x, (want, M) in zip(got[2:], ref[2:]):      # slot (0, 1) names row 3, which is zero
        R.check("gates", x, (want, M), R.sum_tol(n))
    del a, va, got
    torch.cuda.empty_cache()


def test_grouped_linear_without_rows(lib):
    E, K, N = 3, 20, 24
    offsets = torch.zeros(E + 1, dtype=i32, device="cuda")
    v, o = torch.ones(E, N, K, device="cuda"), [Guard(E, N, K), Guard(E, N, K), Guard(E, N), Guard(E, N)]
    grouped_param(lib, E, 0, 0, K, N, 1, p(offsets), None, p(v), p(v), None, None, None, *[x.ptr() for x in o])
    assert all(bool((x.get() == 0).all()) for x in o)


@pytest.mark.parametrize("rows", [6, 300])
def test_grouped_linear_bad_device_data_stays_in_range(lib, rows):
    """Tokens outside the input read as zeros; offsets past the end are cut; nothing outside the tensors is touched."""
    g, K, N = Gen(5), 64, 96
    token = torch.randint(0, rows, (rows,), device="cuda", generator=g.g).to(i32)
    token[0], token[1], token[2] = -1, rows, 2 ** 31 - 1
    offsets = torch.tensor([-5, rows // 2, 2 ** 31 - 1], dtype=i32, device="cuda")
    mw, vw, ma, va = g.n(2, N, K), g.u(2, N, K), g.n(rows, K), g.u(rows, K)
    z, vz = Guard(rows, N), Guard(rows, N)
    grouped_fwd(lib, 2, rows, rows, K, N, 0, p(offsets), p(token), p(mw), p(vw), None, None, p(ma), p(va), z.ptr(), vz.ptr())
    ref = R.grouped_fwd(mw, vw, None, None, ma, va, offsets, token)
    assert bool((z.get()[:3] == 0).all())
    R.check("mu_z", z.get(), ref[0], R.sum_tol(K))
    R.check("var_z", vz.get(), ref[1], R.sum_tol(2 * K))
    o, dm = [Guard(2, N, K) for _ in range(2)], g.n(rows, N)
    grouped_param(lib, 2, rows, rows, K, N, 0, p(offsets), p(token), p(vw), None, p(ma), p(dm), p(dm),
                                      o[0].ptr(), o[1].ptr(), None, None)
    ref = R.grouped_param(vw, None, ma, dm, dm, offsets, token)
    R.check("dmu_w", o[0].get(), ref[0], R.sum_tol(rows))
    R.check("dvar_w", o[1].get(), ref[1], R.sum_tol(rows))


@pytest.mark.parametrize("counts", [[2, 3, 1], [40, 170, 90], [16, 30, 48]])
@pytest.mark.parametrize("K, N", [(200, 96), (199, 97)])
def test_grouped_linear_rows_of_other_experts_do_not_leak(lib, counts, K, N):
    """NaN and infinities in one expert's rows, weights and deltas, and in rows that no expert owns, stay there."""
    g, E = Gen(9), len(counts)
    offsets, S = spread(counts, 3, 4)
    mw, vw, ma, va = g.n(E, N, K, scale=K ** -0.5), g.u(E, N, K, hi=1.0 / K), g.n(S, K), g.u(S, K)
    dm, dv = g.n(S, N), g.n(S, N)
    a, b = int(offsets[1]), int(offsets[2])
    lo, hi = int(offsets[0]), int(offsets[3])
    for t in (ma, va, dm, dv):
        t[a:b], t[:lo], t[hi:] = torch.nan, torch.inf, torch.nan
    mw[1], vw[1] = torch.inf, torch.nan
    z, vz, da, dva = Guard(S, N), Guard(S, N), Guard(S, K), Guard(S, K)
    o = [Guard(E, N, K) for _ in range(2)] + [Guard(E, N) for _ in range(2)]
    vb = g.u(E, N)
    grouped_fwd(lib, E, S, S, K, N, 0, p(offsets), None, p(mw), p(vw), None, None, p(ma), p(va), z.ptr(), vz.ptr())
    grouped_state(lib, E, S, K, N, p(offsets), p(mw), None, p(dm), p(dv), da.ptr(), dva.ptr())
    grouped_param(lib, E, S, S, K, N, 1, p(offsets), None, p(vw), p(vb), p(ma), p(dm), p(dv), *[x.ptr() for x in o])
    rows = torch.cat([torch.arange(lo, a), torch.arange(b, hi)]).cuda()
    for pair, got, L in zip((*R.grouped_fwd(mw, vw, None, None, ma, va, offsets, None), *R.grouped_state(mw, None, dm, dv, offsets)),
                            (z, vz, da, dva), (K, 2 * K, N, N)):
        R.check("rows", got.get(whole=False)[rows], (pair[0][rows], pair[1][rows]), R.sum_tol(L))
    for pair, got in zip(R.grouped_param(vw, vb, ma, dm, dv, offsets, None), o):
        keep = torch.tensor([0, 2], device="cuda")
        R.check("experts", got.get(whole=False)[keep], (pair[0][keep], pair[1][keep]), R.sum_tol(max(counts)))
        assert not bool(torch.isfinite(got.get(whole=False)[1]).any())


@pytest.mark.parametrize("counts", [[5, 7], [30, 12], [100, 64], [300, 140]])
@pytest.mark.parametrize("K, N", [(200, 132), (199, 131)])
def test_grouped_linear_a_row_that_is_not_finite_stays_alone(lib, counts, K, N):
    """One row of each expert holds NaN and infinities: the expert's other rows are what they would be without it."""
    from cutagi_b200 import ops
    g, E = Gen(sum(counts)), len(counts)
    offsets, S = spread(counts)
    mw, vw = g.n(E, N, K, scale=K ** -0.5), g.u(E, N, K, hi=1.0 / K)
    a, va, dm, dv = g.n(S, K), g.u(S, K), g.n(S, N), g.u(S, N)
    clean = (*ops.grouped_linear(mw, vw, None, None, a, va, offsets), *ops.grouped_linear_state(mw, None, dm, dv, offsets))
    bad = offsets[:-1].long() + 3
    for t, x in ((a, torch.nan), (va, torch.inf), (dm, -torch.inf), (dv, torch.nan)):
        t[bad] = x
    rest = torch.ones(S, dtype=torch.bool, device="cuda")
    rest[bad] = False
    dirty = (*ops.grouped_linear(mw, vw, None, None, a, va, offsets), *ops.grouped_linear_state(mw, None, dm, dv, offsets))
    for x, y in zip(clean, dirty):
        assert torch.equal(x[rest], y[rest]) and not bool(torch.isfinite(y[bad]).any())


@pytest.mark.parametrize("rows", [4, 200])
def test_grouped_linear_wide_range_of_values(lib, rows):
    """Entries of one contraction that differ by many powers of two keep the accuracy of 32-bit products: large inputs
    against small weights and the other way round."""
    g, K, N = Gen(11), 128, 64
    scale = torch.exp2(torch.linspace(-30, 30, K, device="cuda"))
    mw, vw = g.n(1, N, K) / scale, g.u(1, N, K, lo=0.1) / scale.square()
    ma, va = g.n(rows, K) * scale, g.u(rows, K, lo=0.1) * scale.square()
    offsets, _ = spread([rows])
    z, vz = Guard(rows, N), Guard(rows, N)
    grouped_fwd(lib, 1, rows, rows, K, N, 0, p(offsets), None, p(mw), p(vw), None, None, p(ma), p(va), z.ptr(), vz.ptr())
    ref = R.grouped_fwd(mw, vw, None, None, ma, va, offsets, None)
    R.check("mu_z", z.get(), ref[0], R.sum_tol(K))
    R.check("var_z", vz.get(), ref[1], R.sum_tol(2 * K))


# -------------------------------------------------------------------------------------------------------------- combine

@pytest.mark.parametrize("T, k, N", [(1, 1, 1), (1, 2, 64), (3, 4, 33), (50, 1, 1000), (17, 8, 1024), (5, 32, 130), (200, 3, 4100), (64, 5, 16)])
@pytest.mark.parametrize("idle, misalign", [(0.0, 0), (0.4, 1), (1.0, 0)])
def test_combine(lib, T, k, N, idle, misalign):
    g = Gen(T + k + N, misalign)
    S = T * k
    pos = torch.randperm(S, device="cuda", generator=g.g).reshape(T, k).to(i32)
    pos[g.u(T, k) < idle] = -1
    if T > 2:
        pos[1, 0], pos[2, 0] = S, -2 ** 31       # names no row
    mg, vg = g.u(T, k), g.u(T, k, hi=0.2)
    mx, vx, dm, dv, jcb = g.n(S, N), g.u(S, N), g.n(T, N), g.u(T, N, lo=-1.0, hi=0.0), g.u(S, N)
    y, vy = Guard(T, N, misalign=misalign), Guard(T, N, misalign=misalign)
    lib.tagi_combine_fwd(T, k, N, S, p(pos), p(mg), p(vg), p(mx), p(vx), y.ptr(), vy.ptr(), st())
    ref = R.combine_fwd(pos, mg, vg, mx, vx)
    R.check("mu_y", y.get(), ref[0], (8 + 2 * k) * R.U)
    R.check("var_y", vy.get(), ref[1], (8 + 2 * k) * R.U)
    for j in (None, jcb):
        dx, dvx, dg, dvg = Guard(S, N, misalign=misalign), Guard(S, N, misalign=misalign), Guard(T, k), Guard(T, k)
        lib.tagi_combine_bwd(T, k, N, S, p(pos), p(mg), p(mx), p(j), p(dm), p(dv), dx.ptr(), dvx.ptr(), dg.ptr(), dvg.ptr(), st())
        ref = R.combine_bwd(pos, mg, mx, j, dm, dv)
        none = torch.isnan(ref[0][0][:, 0])
        for name, got, pair in (("dmu_x", dx, ref[0]), ("dvar_x", dvx, ref[1])):
            t = got.get(whole=False)
            assert bool((t[none] == SENT).all()), "a row that no slot names was written"
            R.check(name, t[~none], (pair[0][~none], pair[1][~none]), 8 * R.U)
        R.check("dmu_g", dg.get(), ref[2], R.sum_tol(N))
        R.check("dvar_g", dvg.get(), ref[3], R.sum_tol(N))
    for j in (None, g.u(T, N)):
        da, dva = Guard(T, N, misalign=misalign), Guard(T, N, misalign=misalign)
        lib.tagi_dispatch_bwd(T, k, N, S, p(pos), p(j), p(mx), p(vx), da.ptr(), dva.ptr(), st())
        ref = R.dispatch_bwd(pos, j, mx, vx)
        R.check("dmu_a", da.get(), ref[0], (8 + 2 * k) * R.U)
        R.check("dvar_a", dva.get(), ref[1], (8 + 2 * k) * R.U)


# ------------------------------------------------------------------------------------------------- streams, graphs, order

def _expert_layer(ops, x):
    r = ops.route(x["s"], x["vs"], 2)
    h, vh = ops.grouped_linear(x["w"], x["vw"], x["b"], x["vb"], x["a"], x["va"], r.offsets, r.token)
    y, vy = ops.combine(r.pos, r.mu_g, r.var_g, h, vh)
    z, vz, m, v = ops.layer_norm(x["g"], x["vg"], None, None, y, vy)
    dm, dv, dg, dvg, _, _ = ops.layer_norm_backward(x["g"], x["vg"], None, y, None, m, v, x["dm"], x["dv"])
    dx, dvx, dmg, dvmg = ops.combine_backward(r.pos, r.mu_g, h, None, dm, dv)
    ds, dvs = ops.route_backward(r, dmg, dvmg)
    dw = ops.grouped_linear_param(x["vw"], x["vb"], x["a"], dx, dvx, r.offsets, r.token)
    dr, dvr = ops.grouped_linear_state(x["w"], None, dx, dvx, r.offsets)
    da, dva = ops.dispatch_backward(r.pos, None, dr, dvr)
    return [z, vz, dg, dvg, ds, dvs, *dw, da, dva]


def _expert_inputs(seed, T=200, E=6, K=96, N=128):
    g = Gen(seed)
    return dict(s=g.n(T, E), vs=g.u(T, E), w=g.n(E, N, K, scale=0.1), vw=g.u(E, N, K, hi=0.01), b=g.n(E, N), vb=g.u(E, N),
                a=g.n(T, K), va=g.u(T, K), g=g.n(N), vg=g.u(N), dm=g.n(T, N), dv=g.u(T, N, lo=-1.0, hi=0.0))


def test_no_tokens_at_all(lib):
    from cutagi_b200 import ops
    out = _expert_layer(ops, _expert_inputs(1, T=0))
    assert [tuple(t.shape) for t in out[:6]] == [(0, 128), (0, 128), (128,), (128,), (0, 6), (0, 6)]
    assert all(not bool(t.any()) for t in out)      # parameter deltas of no tokens are zero


def test_results_repeat_bit_for_bit(lib):
    from cutagi_b200 import ops
    x = _expert_inputs(1)
    first = [t.clone() for t in _expert_layer(ops, x)]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _expert_layer(ops, x)))


@pytest.mark.parametrize("T", [8, 200])
def test_captured_calls_replay_on_new_inputs(lib, T):
    """Two graphs captured from the same calls, replayed at the same time on two streams with inputs that changed (and with
    them the experts' row counts)."""
    from cutagi_b200 import ops
    xs, graphs, outs = [_expert_inputs(i, T) for i in (1, 2)], [], []
    _expert_layer(ops, xs[0])
    torch.cuda.synchronize()
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_expert_layer(ops, x))
        graphs.append(gr)
    for seed in (5, 7):
        want = []
        for i, x in enumerate(xs):
            new = _expert_inputs(seed + i, T)
            for name, t in new.items():
                x[name].copy_(t)
            want.append([t.clone() for t in _expert_layer(ops, new)])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_cut_tiles_repeat_in_graphs_and_beside_each_other(lib):
    """Tiles that are cut along the contraction: the same bits in a graph whose row counts change, twice at the same time."""
    from cutagi_b200 import ops

    def call(x):
        return [*ops.grouped_linear(x["w"], x["vw"], x["b"], x["vb"], x["a"], x["va"], x["o"]),
                *ops.grouped_linear_state(x["w"], None, x["dm"], x["dv"], x["o"]),
                *ops.grouped_linear_param(x["vw"], x["vb"], x["a"], x["dm"], x["dv"], x["o"])]

    def inputs(seed, counts, K=2000, N=1900):
        g = Gen(seed)
        o, S = spread(counts)
        return dict(w=g.n(2, N, K, scale=0.02), vw=g.u(2, N, K, hi=1e-3), b=g.n(2, N), vb=g.u(2, N), a=g.n(S, K), va=g.u(S, K),
                    dm=g.n(S, N), dv=g.u(S, N), o=o)
    xs = [inputs(1, [300, 500]), inputs(2, [700, 100])]
    graphs, outs = [], []
    call(xs[0])
    torch.cuda.synchronize()
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call(x))
        graphs.append(gr)
    for counts in ([60, 740], [0, 800], [400, 400]):
        want = []
        for i, x in enumerate(xs):
            new = inputs(i + 7, counts)
            for name, t in new.items():
                x[name].copy_(t)
            want.append([t.clone() for t in call(new)])
        torch.cuda.synchronize()
        for gr in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                gr.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_calls_follow_the_current_stream(lib):
    """Inputs that are written late on a side stream are seen by calls on that stream, with other calls on a second stream."""
    from cutagi_b200 import ops
    new = [_expert_inputs(3), _expert_inputs(4)]
    want = [[t.clone() for t in _expert_layer(ops, x)] for x in new]
    xs = [{k: torch.full_like(t, torch.nan) for k, t in x.items()} for x in new]
    torch.cuda.synchronize()
    got = []
    for x, n in zip(xs, new):
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda._sleep(20_000_000)
            for k in x:
                x[k].copy_(n[k], non_blocking=True)
            got.append(_expert_layer(ops, x))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# --------------------------------------------------------------------------------------------------- as layers of a network

def _moe_step_reference(layer, r, mu, var, jcb, dm, dv):
    """The expert layer's outputs and deltas in 64 bits, with the kernels' choice of experts."""
    ro, up, dn = layer.router, layer.up, layer.down
    off1 = torch.tensor([0, mu.shape[0]], device="cuda")
    one = lambda t: t[None]  # noqa: E731
    (s, _), (vs, _) = R.grouped_fwd(one(ro.mu_w), one(ro.var_w), one(ro.mu_b), one(ro.var_b), mu, var, off1, None)
    expert, (g, _), (vg, _), *_ = R.route_fwd(s, vs, layer.top_k)
    assert torch.equal(expert, r.expert.long())
    (h, _), (vh, _) = R.grouped_fwd(up.mu_w, up.var_w, up.mu_b, up.var_b, mu, var, r.offsets, r.token)
    j = (h > 0).double()
    h, vh = h * j, vh * j
    (x, _), (vx, _) = R.grouped_fwd(dn.mu_w, dn.var_w, dn.mu_b, dn.var_b, h, vh, r.offsets, None)
    y = R.combine_fwd(r.pos, g, vg, x, vx)
    dx, dvx, dg, dvg = [t[0] for t in R.combine_bwd(r.pos, g, x, None, dm, dv)]
    ds, dvs = [t[0] for t in R.route_bwd(r.expert, g, dg, dvg, s.shape[1])]
    pd = R.grouped_param(dn.var_w, dn.var_b, h, dx, dvx, r.offsets, None)
    dh, dvh = [t[0] for t in R.grouped_state(dn.mu_w, j, dx, dvx, r.offsets)]
    pu = R.grouped_param(up.var_w, up.var_b, mu, dh, dvh, r.offsets, r.token)
    dr, dvr = [t[0] for t in R.grouped_state(up.mu_w, None, dh, dvh, r.offsets)]
    da, dva = [t[0] for t in R.dispatch_bwd(r.pos, jcb, dr, dvr)]
    pr = R.grouped_param(one(ro.var_w), one(ro.var_b), mu, ds, dvs, off1, None)
    ra, rva = [t[0] for t in R.grouped_state(one(ro.mu_w), jcb, ds, dvs, off1)]
    return y[0][0], y[1][0], da + ra, dva + rva, [q[0] for q in pd + pu] + [q[0][0] for q in pr]


@pytest.mark.parametrize("T", [3, 150])
def test_mixture_of_experts_layer(lib, T):
    from cutagi_b200 import nn
    layer = nn.MixtureOfExperts(48, 96, 40, 5, 2, seed=3)
    layer.init_shape((48,))
    g = Gen(T)
    mu, var, jcb, dm, dv = g.n(T, 48), g.u(T, 48, hi=0.1), (g.u(T, 48) < 0.7).float(), g.n(T, 40), g.u(T, 40, lo=-0.1, hi=0.0)
    y, vy, _ = layer.forward(mu, var, jcb)
    da, dva = layer.backward(dm, dv)
    ref = _moe_step_reference(layer, layer.saved[0], mu, var, jcb, dm, dv)
    got = [y, vy, da, dva] + layer.delta_tensors()
    want = [*ref[:4], *ref[4]]
    assert len(got) == len(want)
    # three layers in a row, each within (16 + 4 sqrt(96)) U of its magnitudes: 1e-5 of the largest entry leaves room for
    # sums that cancel (the network-level tests of the Linear layers ask for the same)
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= 1e-5 * b.abs().max()


def test_token_network_trains_and_reloads(lib):
    """LayerNorm and an expert layer inside a Sequential: steps, packed deltas and a reloaded state give the same bits."""
    import numpy as np
    from cutagi_b200 import nn
    spec = [("linear", 12, 32, True), ("relu",), ("ln", 32), ("moe", 32, 64, 24, 4, 2, True), ("ln", 24), ("linear", 24, 3, True)]
    rng = np.random.default_rng(0)
    x, t = rng.standard_normal((64, 12)).astype("f"), rng.standard_normal((64, 3)).astype("f")

    def train(net, steps):
        up = nn.OutputUpdater()
        for _ in range(steps):
            net.forward(x)
            up.update(net, t, np.full_like(t, 0.1))
            net.backward()
            net.step()
        return net.state_dict()
    a, b = nn.build(spec, (12,), seed=1), nn.build(spec, (12,), seed=1)
    b.pack_deltas()
    sa, sb = train(a, 3), train(b, 3)
    assert set(sa) == {"Linear.0", "LayerNorm.2", "MixtureOfExperts.3.router", "MixtureOfExperts.3.up", "MixtureOfExperts.3.down",
                       "LayerNorm.4", "Linear.5"}
    first = nn.build(spec, (12,), seed=1).state_dict()
    for k in sa:
        for u, v, w in zip(sa[k], sb[k], first[k]):
            assert np.array_equal(u, v) and np.isfinite(u).all() and not np.array_equal(u, w), k
    c = nn.build(spec, (12,), seed=2)
    c.load_state_dict(sa)
    a.eval(), c.eval()
    assert all(torch.equal(u, v) for u, v in zip(a.forward(x), c.forward(x)))


def test_expert_layer_errors(lib):
    from cutagi_b200 import nn, ops
    with pytest.raises(ValueError):
        nn.MixtureOfExperts(8, 8, 8, 2, 3)
    with pytest.raises(RuntimeError):
        nn.Sequential(nn.Linear(8, 4), nn.LayerNorm(5))
    with pytest.raises(RuntimeError):
        nn.Sequential(nn.Linear(8, 4), nn.MixtureOfExperts(5, 8, 8, 2, 1))
    z = torch.zeros(6, 8, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        ops.layer_norm(z[0], z[0], None, None, torch.zeros(8, 6, device="cuda").t(), z)
    with pytest.raises(ValueError, match="expected"):
        ops.layer_norm(z[0].double(), z[0], None, None, z, z)
    with pytest.raises(ValueError, match="k: "):
        ops.route(z, z, 9)
