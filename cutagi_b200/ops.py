"""The layers of token models on torch tensors: LayerNorm, expert routing, Linear layers grouped by expert and the
combination of the experts' rows. Each function allocates its outputs, calls the entry point of ``include/tagi_b200.h`` with
the same name on the tensors' device and its current stream, and returns the outputs; the header states the formulas.
Tensors must be contiguous float32 (indices: int32) on one CUDA device.
"""
from typing import NamedTuple, Optional

import torch

from . import capi

_F, _I = torch.float32, torch.int32
_MOST = 2 ** 31 - 1   # the entry points' sizes are 32-bit integers, which ctypes would cut without a word
# what torch.cuda.current_stream and current_device come down to
_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _run(name, index, *args):
    """Calls the entry point with device `index` current, on its current stream; raises TagiError on a bad status."""
    if index != _device():
        with torch.cuda.device(index):
            return _run(name, index, *args)
    lib = capi.load()
    rc = getattr(lib, name)(*args, _stream(index))
    if rc != capi.TAGI_OK:
        raise capi.TagiError(rc, lib.tagi_last_error_string().decode())


def _index(name, t, dim=2):
    """The CUDA device of the tensor that the others have to share, after a look at its number of dimensions."""
    if t.dim() != dim:
        raise ValueError(f"{name}: expected a tensor of {'two dimensions' if dim == 2 else f'{dim} dimensions'}, got {tuple(t.shape)}")
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name}: expected a tensor on a CUDA device, got {t.device}")
    if t.numel() > _MOST and max(t.shape) > _MOST:
        raise ValueError(f"{name}: more than 2^31 - 1 entries along a dimension: {tuple(t.shape)}")
    return index


def _rows(name, n):
    if n > _MOST:
        raise ValueError(f"{name}: more than 2^31 - 1 rows: {n}")
    return n


def _p(name, t, shape, index, dtype=_F):
    """The tensor's address (None for None); raises ValueError where it is not what the kernels read."""
    if t is None:
        return None
    if t.dtype is dtype and t.get_device() == index and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{index}, got {t.dtype} "
                     f"{tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")


def _pair(name, a, b):
    if (a is None) != (b is None):
        raise ValueError(f"{name}: both of the pair or neither")
    return int(a is not None)


def _two(like, *shape):
    """Two float tensors of the shape (without one: of like's) on like's device. The launch latency of a small call is that of
    its allocations: these are the cheap forms."""
    if shape:
        return like.new_empty(*shape), like.new_empty(*shape)
    return torch.empty_like(like), torch.empty_like(like)


def _workspace(nbytes, like):
    """(tensor that keeps the memory, address)"""
    if nbytes == 0:
        return None, None
    t = like.new_empty((nbytes + 3) // 4)
    return t, t.data_ptr()


def layer_norm(mu_w, var_w, mu_b, var_b, mu_a, var_a, eps=1e-5):
    """tagi_ln_fwd on rows [R][n]: (mu_z, var_z, mu_row, var_row)."""
    bias, i = _pair("mu_b / var_b", mu_b, var_b), _index("mu_a", mu_a)
    R, n = s = mu_a.shape
    f = (n,)
    inputs = (_p("mu_w", mu_w, f, i), _p("var_w", var_w, f, i), _p("mu_b", mu_b, f, i), _p("var_b", var_b, f, i),
              _p("mu_a", mu_a, s, i), _p("var_a", var_a, s, i))
    (mu_z, var_z), (mu_row, var_row) = _two(mu_a), _two(mu_a, R)
    _run("tagi_ln_fwd", i, R, n, bias, eps, *inputs, mu_row.data_ptr(), var_row.data_ptr(), mu_z.data_ptr(), var_z.data_ptr())
    return mu_z, var_z, mu_row, var_row


def layer_norm_backward(mu_w, var_w, var_b, mu_a, jcb, mu_row, var_row, dmu_o, dvar_o, eps=1e-5, state_update=True, out=None):
    """tagi_ln_bwd: (dmu, dvar, dmu_w, dvar_w, dmu_b, dvar_b); dmu and dvar are None without state_update, the bias deltas
    without var_b. `out`: the four tensors that receive the parameter deltas (None where there is no bias)."""
    i = _index("mu_a", mu_a)
    R, n = s = mu_a.shape
    f, bias = (n,), var_b is not None
    inputs = (_p("mu_w", mu_w, f, i), _p("var_w", var_w, f, i), _p("var_b", var_b, f, i), _p("mu_a", mu_a, s, i),
              _p("jcb", jcb, s, i), _p("mu_row", mu_row, (R,), i), _p("var_row", var_row, (R,), i), _p("dmu_o", dmu_o, s, i),
              _p("dvar_o", dvar_o, s, i))
    if out is None:
        out = mu_w.new_empty(4 if bias else 2, n).unbind(0)
        outputs = [t.data_ptr() for t in out] if bias else (out[0].data_ptr(), out[1].data_ptr(), None, None)
        out = out if bias else (*out, None, None)
    else:
        outputs = [_p(f"out[{k}]", t, f, i) for k, t in enumerate(out)]
    dmu, dvar = _two(mu_a) if state_update else (None, None)
    state = (dmu.data_ptr(), dvar.data_ptr()) if state_update else (None, None)
    nbytes = capi.load().tagi_ln_bwd_workspace_bytes(R, n)
    keep, ws = _workspace(nbytes, mu_a)
    _run("tagi_ln_bwd", i, R, n, int(bias), int(state_update), eps, *inputs, *state, *outputs, ws, nbytes)
    return (dmu, dvar, *out)


class Routing(NamedTuple):
    """What tagi_route_fwd writes: [T][k] experts, gate moments and rows of the slots; the dispatch order of the rows."""
    expert: torch.Tensor
    mu_g: torch.Tensor
    var_g: torch.Tensor
    offsets: torch.Tensor
    token: torch.Tensor
    pos: torch.Tensor
    experts: int


def route(mu_s, var_s: Optional[torch.Tensor], k) -> Routing:
    """tagi_route_fwd: the k best of the E experts for each token by its scores [T][E]."""
    i = _index("mu_s", mu_s)
    T, E = s = mu_s.shape
    if not 1 <= k <= E:
        raise ValueError(f"k: expected 1 to {E} (the number of experts), got {k}")
    inputs = _p("mu_s", mu_s, s, i), _p("var_s", var_s, s, i)
    mu_g, var_g = _two(mu_s, T, k)
    expert, pos = torch.empty_like(mu_g, dtype=_I), torch.empty_like(mu_g, dtype=_I)
    offsets, token = mu_s.new_empty(E + 1, dtype=_I), mu_s.new_empty(T * k, dtype=_I)
    nbytes = capi.load().tagi_route_workspace_bytes(T, E, k)
    keep, ws = _workspace(nbytes, mu_s)
    _run("tagi_route_fwd", i, T, E, k, *inputs, expert.data_ptr(), mu_g.data_ptr(), var_g.data_ptr(), offsets.data_ptr(),
         token.data_ptr(), pos.data_ptr(), ws, nbytes)
    return Routing(expert, mu_g, var_g, offsets, token, pos, E)


def route_backward(r: Routing, dmu_g, dvar_g):
    """tagi_route_bwd: the deltas of the scores, (dmu_s, dvar_s) [T][E]."""
    i, s = _index("expert", r.expert), r.expert.shape
    T, k = s
    dmu_s, dvar_s = _two(r.mu_g, T, r.experts)
    _run("tagi_route_bwd", i, T, r.experts, k, _p("expert", r.expert, s, i, _I), _p("mu_g", r.mu_g, s, i), _p("dmu_g", dmu_g, s, i),
         _p("dvar_g", dvar_g, s, i), dmu_s.data_ptr(), dvar_s.data_ptr())
    return dmu_s, dvar_s


def grouped_linear(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, token=None):
    """tagi_grouped_linear_fwd: (mu_z, var_z) [S][N] in dispatch order. `token` (int32 [S]): the row of mu_a that each row
    reads; without it row p reads row p. Rows that no expert owns are not written."""
    i, (E, N, K), R = _index("mu_w", mu_w, 3), mu_w.shape, _rows("mu_a", mu_a.shape[0])
    S = R if token is None else _rows("token", token.numel())
    bias, w, b = _pair("mu_b / var_b", mu_b, var_b), mu_w.shape, (E, N)
    inputs = (_p("offsets", offsets, (E + 1,), i, _I), _p("token", token, (S,), i, _I), _p("mu_w", mu_w, w, i), _p("var_w", var_w, w, i),
              _p("mu_b", mu_b, b, i), _p("var_b", var_b, b, i), _p("mu_a", mu_a, (R, K), i), _p("var_a", var_a, (R, K), i))
    mu_z, var_z = _two(mu_w, S, N)
    nbytes = capi.load().tagi_grouped_linear_workspace_bytes(0, E, S, R, K, N)
    keep, ws = _workspace(nbytes, mu_w)
    _run("tagi_grouped_linear_fwd", i, E, S, R, K, N, bias, *inputs, mu_z.data_ptr(), var_z.data_ptr(), ws, nbytes)
    return mu_z, var_z


def grouped_linear_state(mu_w, jcb, dmu_z, dvar_z, offsets):
    """tagi_grouped_linear_bwd_state: (dmu_a, dvar_a) [S][K] in dispatch order."""
    i, (E, N, K), S = _index("mu_w", mu_w, 3), mu_w.shape, _rows("dmu_z", dmu_z.shape[0])
    inputs = (_p("offsets", offsets, (E + 1,), i, _I), _p("mu_w", mu_w, mu_w.shape, i), _p("jcb", jcb, (S, K), i),
              _p("dmu_z", dmu_z, (S, N), i), _p("dvar_z", dvar_z, (S, N), i))
    dmu_a, dvar_a = _two(mu_w, S, K)
    nbytes = capi.load().tagi_grouped_linear_workspace_bytes(1, E, S, S, K, N)
    keep, ws = _workspace(nbytes, mu_w)
    _run("tagi_grouped_linear_bwd_state", i, E, S, K, N, *inputs, dmu_a.data_ptr(), dvar_a.data_ptr(), ws, nbytes)
    return dmu_a, dvar_a


def grouped_linear_param(var_w, var_b, mu_a, dmu_z, dvar_z, offsets, token=None, out=None):
    """tagi_grouped_linear_bwd_param: (dmu_w, dvar_w, dmu_b, dvar_b), the bias deltas None without var_b. `out`: the four
    tensors that receive them."""
    i, w = _index("var_w", var_w, 3), var_w.shape
    (E, N, K), R, S = w, _rows("mu_a", mu_a.shape[0]), _rows("dmu_z", dmu_z.shape[0])
    bias, b = var_b is not None, (E, N)
    inputs = (_p("offsets", offsets, (E + 1,), i, _I), _p("token", token, (S,), i, _I), _p("var_w", var_w, w, i), _p("var_b", var_b, b, i),
              _p("mu_a", mu_a, (R, K), i), _p("dmu_z", dmu_z, (S, N), i), _p("dvar_z", dvar_z, (S, N), i))
    if out is None:
        out = (*_two(var_w), *(_two(var_b) if bias else (None, None)))
        outputs = [None if t is None else t.data_ptr() for t in out]
    else:
        outputs = [_p(f"out[{k}]", t, w if k < 2 else b, i) for k, t in enumerate(out)]
    nbytes = capi.load().tagi_grouped_linear_workspace_bytes(2, E, S, R, K, N)
    keep, ws = _workspace(nbytes, var_w)
    _run("tagi_grouped_linear_bwd_param", i, E, S, R, K, N, int(bias), *inputs, *outputs, ws, nbytes)
    return tuple(out)


def combine(pos, mu_g, var_g, mu_x, var_x):
    """tagi_combine_fwd: (mu_y, var_y) [T][N] from the experts' rows mu_x / var_x [S][N]."""
    i, s, x = _index("pos", pos), pos.shape, mu_x.shape
    _index("mu_x", mu_x)
    (T, k), (S, N) = s, x
    inputs = (_p("pos", pos, s, i, _I), _p("mu_g", mu_g, s, i), _p("var_g", var_g, s, i), _p("mu_x", mu_x, x, i), _p("var_x", var_x, x, i))
    mu_y, var_y = _two(mu_x, T, N)
    _run("tagi_combine_fwd", i, T, k, N, S, *inputs, mu_y.data_ptr(), var_y.data_ptr())
    return mu_y, var_y


def combine_backward(pos, mu_g, mu_x, jcb, dmu_y, dvar_y):
    """tagi_combine_bwd: (dmu_x, dvar_x [S][N], dmu_g, dvar_g [T][k])."""
    i, s, x = _index("pos", pos), pos.shape, mu_x.shape
    _index("mu_x", mu_x)
    (T, k), (S, N) = s, x
    inputs = (_p("pos", pos, s, i, _I), _p("mu_g", mu_g, s, i), _p("mu_x", mu_x, x, i), _p("jcb", jcb, x, i), _p("dmu_y", dmu_y, (T, N), i),
              _p("dvar_y", dvar_y, (T, N), i))
    (dmu_x, dvar_x), (dmu_g, dvar_g) = _two(mu_x), _two(mu_g)
    _run("tagi_combine_bwd", i, T, k, N, S, *inputs, dmu_x.data_ptr(), dvar_x.data_ptr(), dmu_g.data_ptr(), dvar_g.data_ptr())
    return dmu_x, dvar_x, dmu_g, dvar_g


def dispatch_backward(pos, jcb, dmu_x, dvar_x):
    """tagi_dispatch_bwd: (dmu_a, dvar_a) [T][N] of the tokens from the deltas of their rows."""
    i, s, x = _index("pos", pos), pos.shape, dmu_x.shape
    _index("dmu_x", dmu_x)
    (T, k), (S, N) = s, x
    inputs = _p("pos", pos, s, i, _I), _p("jcb", jcb, (T, N), i), _p("dmu_x", dmu_x, x, i), _p("dvar_x", dvar_x, x, i)
    dmu_a, dvar_a = _two(dmu_x, T, N)
    _run("tagi_dispatch_bwd", i, T, k, N, S, *inputs, dmu_a.data_ptr(), dvar_a.data_ptr())
    return dmu_a, dvar_a
