"""The layers of token models on torch tensors: LayerNorm, expert routing, Linear layers grouped by expert and the
combination of the experts' rows. Each function allocates its outputs, calls the entry point of ``include/tagi_b200.h`` with
the same name on the tensors' device and its current stream, and returns the outputs; the header states the formulas.
Tensors must be contiguous float32 (indices: int32) on one CUDA device.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import capi

_F, _I = torch.float32, torch.int32


def _run(name, device, *args):
    """Calls the entry point with `device` current, on its current stream; raises TagiError on a bad status."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _run(name, device, *args)
    lib = capi.load()
    rc = getattr(lib, name)(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc != capi.TAGI_OK:
        raise capi.TagiError(rc, lib.tagi_last_error_string().decode())


def _check(device, **tensors):
    """name=(tensor or None, shape, dtype): raises ValueError where a tensor is not what the kernels read."""
    for name, (t, shape, dtype) in tensors.items():
        if t is None:
            continue
        if t.dtype != dtype or t.device != device or t.device.type != "cuda":
            raise ValueError(f"{name}: expected {dtype} on {device} (a CUDA device), got {t.dtype} on {t.device}")
        if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
            raise ValueError(f"{name}: expected a contiguous tensor of shape {tuple(shape)}, got {tuple(t.shape)}"
                             f"{'' if t.is_contiguous() else ' (not contiguous)'}")


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(name, t):
    if t.dim() != 2:
        raise ValueError(f"{name}: expected a tensor of two dimensions, got {tuple(t.shape)}")
    return t.shape


def _pair(name, a, b):
    if (a is None) != (b is None):
        raise ValueError(f"{name}: both of the pair or neither")
    return int(a is not None)


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def layer_norm(mu_w, var_w, mu_b, var_b, mu_a, var_a, eps=1e-5):
    """tagi_ln_fwd on rows [R][n]: (mu_z, var_z, mu_row, var_row)."""
    R, n = _rows("mu_a", mu_a)
    d = mu_a.device
    bias = _pair("mu_b / var_b", mu_b, var_b)
    _check(d, mu_a=(mu_a, (R, n), _F), var_a=(var_a, (R, n), _F), mu_w=(mu_w, (n,), _F), var_w=(var_w, (n,), _F),
           mu_b=(mu_b, (n,), _F), var_b=(var_b, (n,), _F))
    mu_z, var_z = torch.empty_like(mu_a), torch.empty_like(mu_a)
    stats = torch.empty(2, R, dtype=_F, device=d)
    _run("tagi_ln_fwd", d, R, n, bias, C.c_float(eps), _p(mu_w), _p(var_w), _p(mu_b), _p(var_b), _p(mu_a), _p(var_a),
         _p(stats[0]), _p(stats[1]), _p(mu_z), _p(var_z))
    return mu_z, var_z, stats[0], stats[1]


def layer_norm_backward(mu_w, var_w, var_b, mu_a, jcb, mu_row, var_row, dmu_o, dvar_o, eps=1e-5, state_update=True, out=None):
    """tagi_ln_bwd: (dmu, dvar, dmu_w, dvar_w, dmu_b, dvar_b); dmu and dvar are None without state_update, the bias deltas
    without var_b. `out`: the four tensors that receive the parameter deltas (None where there is no bias)."""
    R, n = _rows("mu_a", mu_a)
    d = mu_a.device
    bias = var_b is not None
    _check(d, mu_a=(mu_a, (R, n), _F), jcb=(jcb, (R, n), _F), dmu_o=(dmu_o, (R, n), _F), dvar_o=(dvar_o, (R, n), _F),
           mu_w=(mu_w, (n,), _F), var_w=(var_w, (n,), _F), var_b=(var_b, (n,), _F), mu_row=(mu_row, (R,), _F),
           var_row=(var_row, (R,), _F))
    if out is None:
        out = [torch.empty(n, dtype=_F, device=d) if b else None for b in (True, True, bias, bias)]
    else:
        _check(d, **{f"out[{i}]": (t, (n,), _F) for i, t in enumerate(out)})
    dmu, dvar = (torch.empty_like(mu_a), torch.empty_like(mu_a)) if state_update else (None, None)
    nbytes = capi.load().tagi_ln_bwd_workspace_bytes(R, n)
    ws = _workspace(nbytes, d)
    _run("tagi_ln_bwd", d, R, n, int(bias), int(state_update), C.c_float(eps), _p(mu_w), _p(var_w), _p(var_b), _p(mu_a),
         _p(jcb), _p(mu_row), _p(var_row), _p(dmu_o), _p(dvar_o), _p(dmu), _p(dvar), *[_p(t) for t in out], _p(ws), nbytes)
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
    T, E = _rows("mu_s", mu_s)
    d = mu_s.device
    _check(d, mu_s=(mu_s, (T, E), _F), var_s=(var_s, (T, E), _F))
    if not 1 <= k <= E:
        raise ValueError(f"k: expected 1 to {E} (the number of experts), got {k}")
    expert, pos = torch.empty(2, T, k, dtype=_I, device=d)
    mu_g, var_g = torch.empty(2, T, k, dtype=_F, device=d)
    offsets, token = torch.empty(E + 1, dtype=_I, device=d), torch.empty(T * k, dtype=_I, device=d)
    nbytes = capi.load().tagi_route_workspace_bytes(T, E, k)
    ws = _workspace(nbytes, d)
    _run("tagi_route_fwd", d, T, E, k, _p(mu_s), _p(var_s), _p(expert), _p(mu_g), _p(var_g), _p(offsets), _p(token), _p(pos),
         _p(ws), nbytes)
    return Routing(expert, mu_g, var_g, offsets, token, pos, E)


def route_backward(r: Routing, dmu_g, dvar_g):
    """tagi_route_bwd: the deltas of the scores, (dmu_s, dvar_s) [T][E]."""
    T, k = _rows("expert", r.expert)
    d = r.expert.device
    _check(d, expert=(r.expert, (T, k), _I), mu_g=(r.mu_g, (T, k), _F), dmu_g=(dmu_g, (T, k), _F), dvar_g=(dvar_g, (T, k), _F))
    dmu_s, dvar_s = torch.empty(2, T, r.experts, dtype=_F, device=d)
    _run("tagi_route_bwd", d, T, r.experts, k, _p(r.expert), _p(r.mu_g), _p(dmu_g), _p(dvar_g), _p(dmu_s), _p(dvar_s))
    return dmu_s, dvar_s


def _weights(name, w):
    if w.dim() != 3:
        raise ValueError(f"{name}: expected [experts][outputs][inputs], got {tuple(w.shape)}")
    return w.shape


def grouped_linear(mu_w, var_w, mu_b, var_b, mu_a, var_a, offsets, token=None):
    """tagi_grouped_linear_fwd: (mu_z, var_z) [S][N] in dispatch order. `token` (int32 [S]): the row of mu_a that each row
    reads; without it row p reads row p. Rows that no expert owns are not written."""
    E, N, K = _weights("mu_w", mu_w)
    R, S = mu_a.shape[0], mu_a.shape[0] if token is None else token.numel()
    d = mu_a.device
    bias = _pair("mu_b / var_b", mu_b, var_b)
    _check(d, mu_w=(mu_w, (E, N, K), _F), var_w=(var_w, (E, N, K), _F), mu_b=(mu_b, (E, N), _F), var_b=(var_b, (E, N), _F),
           mu_a=(mu_a, (R, K), _F), var_a=(var_a, (R, K), _F), offsets=(offsets, (E + 1,), _I), token=(token, (S,), _I))
    mu_z, var_z = torch.empty(2, S, N, dtype=_F, device=d)
    nbytes = capi.load().tagi_grouped_linear_workspace_bytes(S, R, K)
    ws = _workspace(nbytes, d)
    _run("tagi_grouped_linear_fwd", d, E, S, R, K, N, bias, _p(offsets), _p(token), _p(mu_w), _p(var_w), _p(mu_b), _p(var_b),
         _p(mu_a), _p(var_a), _p(mu_z), _p(var_z), _p(ws), nbytes)
    return mu_z, var_z


def grouped_linear_state(mu_w, jcb, dmu_z, dvar_z, offsets):
    """tagi_grouped_linear_bwd_state: (dmu_a, dvar_a) [S][K] in dispatch order."""
    E, N, K = _weights("mu_w", mu_w)
    S, d = dmu_z.shape[0], dmu_z.device
    _check(d, mu_w=(mu_w, (E, N, K), _F), jcb=(jcb, (S, K), _F), dmu_z=(dmu_z, (S, N), _F), dvar_z=(dvar_z, (S, N), _F),
           offsets=(offsets, (E + 1,), _I))
    dmu_a, dvar_a = torch.empty(2, S, K, dtype=_F, device=d)
    _run("tagi_grouped_linear_bwd_state", d, E, S, K, N, _p(offsets), _p(mu_w), _p(jcb), _p(dmu_z), _p(dvar_z), _p(dmu_a),
         _p(dvar_a))
    return dmu_a, dvar_a


def grouped_linear_param(var_w, var_b, mu_a, dmu_z, dvar_z, offsets, token=None, out=None):
    """tagi_grouped_linear_bwd_param: (dmu_w, dvar_w, dmu_b, dvar_b), the bias deltas None without var_b. `out`: the four
    tensors that receive them."""
    E, N, K = _weights("var_w", var_w)
    R, S, d = mu_a.shape[0], dmu_z.shape[0], dmu_z.device
    bias = var_b is not None
    _check(d, var_w=(var_w, (E, N, K), _F), var_b=(var_b, (E, N), _F), mu_a=(mu_a, (R, K), _F), dmu_z=(dmu_z, (S, N), _F),
           dvar_z=(dvar_z, (S, N), _F), offsets=(offsets, (E + 1,), _I), token=(token, (S,), _I))
    if out is None:
        out = [torch.empty_like(var_w), torch.empty_like(var_w)] + [torch.empty_like(var_b) if bias else None for _ in range(2)]
    else:
        _check(d, **{f"out[{i}]": (t, (E, N, K) if i < 2 else (E, N), _F) for i, t in enumerate(out)})
    _run("tagi_grouped_linear_bwd_param", d, E, S, R, K, N, int(bias), _p(offsets), _p(token), _p(var_w), _p(var_b), _p(mu_a),
         _p(dmu_z), _p(dvar_z), *[_p(t) for t in out])
    return tuple(out)


def combine(pos, mu_g, var_g, mu_x, var_x):
    """tagi_combine_fwd: (mu_y, var_y) [T][N] from the experts' rows mu_x / var_x [S][N]."""
    (T, k), (S, N), d = _rows("pos", pos), _rows("mu_x", mu_x), pos.device
    _check(d, pos=(pos, (T, k), _I), mu_g=(mu_g, (T, k), _F), var_g=(var_g, (T, k), _F), mu_x=(mu_x, (S, N), _F),
           var_x=(var_x, (S, N), _F))
    mu_y, var_y = torch.empty(2, T, N, dtype=_F, device=d)
    _run("tagi_combine_fwd", d, T, k, N, S, _p(pos), _p(mu_g), _p(var_g), _p(mu_x), _p(var_x), _p(mu_y), _p(var_y))
    return mu_y, var_y


def combine_backward(pos, mu_g, mu_x, jcb, dmu_y, dvar_y):
    """tagi_combine_bwd: (dmu_x, dvar_x [S][N], dmu_g, dvar_g [T][k])."""
    (T, k), (S, N), d = _rows("pos", pos), _rows("mu_x", mu_x), pos.device
    _check(d, pos=(pos, (T, k), _I), mu_g=(mu_g, (T, k), _F), mu_x=(mu_x, (S, N), _F), jcb=(jcb, (S, N), _F),
           dmu_y=(dmu_y, (T, N), _F), dvar_y=(dvar_y, (T, N), _F))
    dmu_x, dvar_x = torch.empty(2, S, N, dtype=_F, device=d)
    dmu_g, dvar_g = torch.empty(2, T, k, dtype=_F, device=d)
    _run("tagi_combine_bwd", d, T, k, N, S, _p(pos), _p(mu_g), _p(mu_x), _p(jcb), _p(dmu_y), _p(dvar_y), _p(dmu_x), _p(dvar_x),
         _p(dmu_g), _p(dvar_g))
    return dmu_x, dvar_x, dmu_g, dvar_g


def dispatch_backward(pos, jcb, dmu_x, dvar_x):
    """tagi_dispatch_bwd: (dmu_a, dvar_a) [T][N] of the tokens from the deltas of their rows."""
    (T, k), (S, N), d = _rows("pos", pos), _rows("dmu_x", dmu_x), pos.device
    _check(d, pos=(pos, (T, k), _I), jcb=(jcb, (T, N), _F), dmu_x=(dmu_x, (S, N), _F), dvar_x=(dvar_x, (S, N), _F))
    dmu_a, dvar_a = torch.empty(2, T, N, dtype=_F, device=d)
    _run("tagi_dispatch_bwd", d, T, k, N, S, _p(pos), _p(jcb), _p(dmu_x), _p(dvar_x), _p(dmu_a), _p(dvar_a))
    return dmu_a, dvar_a
