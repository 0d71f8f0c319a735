"""The operators of token models on (mean, variance) tensors, as cases that can be timed and compared: layer norm, expert
routing, Linear layers grouped by expert, and the combination of the experts' outputs.

``own`` selects how a pass is computed: False, in elementary torch operations; True, by the library's entry points.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5


def listed():
    return [
        # one token on its way through a served network: latency of a single launch
        dict(name="ln_fwd_token", op="ln_fwd", rows=1, n=4096, bias=True),
        # the norm in front of a layer of a training batch: 16384 tokens
        dict(name="ln_fwd_batch", op="ln_fwd", rows=16384, n=4096, bias=True),
        # its backward pass behind a ReLU: state deltas and the four parameter deltas
        dict(name="ln_bwd_batch", op="ln_bwd", rows=8192, n=2048, bias=True, jcb=True),
        # routing of a handful of tokens while serving
        dict(name="route_few", op="route", tokens=4, experts=8, k=2, barred=0.0, train=False),
        # routing of a training batch over many experts with the router's deltas; some experts barred, some tokens wholly
        dict(name="route_batch", op="route", tokens=32768, experts=128, k=8, barred=0.05, train=True),
        # one token through its two experts: two weight matrices are read once
        dict(name="grouped_fwd_token", op="grouped_fwd", tokens=1, experts=8, k=2, K=4096, N=4096, bias=True, skew=0.0),
        # a serving batch spread thin over many experts: a few rows for each weight matrix
        dict(name="grouped_fwd_serve", op="grouped_fwd", tokens=256, experts=64, k=4, K=1024, N=1024, bias=True, skew=0.5),
        # a training batch: 8192 rows over eight experts of the 4096 x 4096 layer, unevenly
        dict(name="grouped_fwd_batch", op="grouped_fwd", tokens=4096, experts=8, k=2, K=4096, N=4096, bias=True, skew=0.5),
        # the state pass at sizes that no tile divides
        dict(name="grouped_state_odd", op="grouped_state", tokens=1501, experts=5, k=2, K=1001, N=1515, skew=1.0),
        # the parameter pass of a training batch; its input rows are gathered from the tokens
        dict(name="grouped_param_batch", op="grouped_param", tokens=4096, experts=8, k=2, K=1024, N=4096, bias=True, skew=0.5),
        # the experts' outputs joined for each token
        dict(name="combine_fwd_batch", op="combine_fwd", tokens=16384, k=2, N=2048, idle=0.0),
        # and its backward pass, with the deltas of the gates; some slots have no expert
        dict(name="combine_bwd_batch", op="combine_bwd", tokens=8192, k=4, N=1001, idle=0.05),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "route", "grouped_fwd", "grouped_fwd", "grouped_state", "grouped_param",
                     "combine_fwd", "combine_bwd", "dispatch_bwd"])
    if op in ("ln_fwd", "ln_bwd"):
        n = _log(rng, 2, 8192)
        c = dict(op=op, rows=_log(rng, 1, min(16384, (1 << 25) // n)), n=n, bias=rng.random() < 0.8)
        return dict(c, jcb=rng.random() < 0.5) if op == "ln_bwd" else c
    if op == "route":
        experts = _log(rng, 2, 256)
        return dict(op=op, tokens=_log(rng, 1, min(32768, (1 << 22) // experts)), experts=experts,
                    k=rng.randint(1, min(8, experts)), barred=rng.choice([0.0, 0.05, 0.5]), train=rng.random() < 0.6)
    if op.startswith("grouped"):
        experts = _log(rng, 1, 64)
        K, N = _log(rng, 16, 4096), _log(rng, 16, 4096)
        while experts * K * N > 1 << 27:
            experts = max(1, experts // 2)
        k = rng.randint(1, min(4, experts))
        most = max(1, min(8192, (1 << 36) // (K * N * k)))
        c = dict(op=op, tokens=_log(rng, 1, most), experts=experts, k=k, K=K, N=N, skew=rng.choice([0.0, 0.5, 2.0]))
        return c if op == "grouped_state" else dict(c, bias=rng.random() < 0.8)
    k, N = rng.randint(1, 8), _log(rng, 16, 4096)
    c = dict(op=op, tokens=_log(rng, 1, min(16384, (1 << 25) // (k * N))), k=k, N=N, idle=rng.choice([0.0, 0.05, 0.5]))
    return dict(c, jcb=rng.random() < 0.5) if op == "dispatch_bwd" else c


# ------------------------------------------------------------------------------------------------------------- inputs

class _Gen:
    """Tensors of one seed, in the order in which they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=self.g).mul_(scale)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device="cuda", generator=self.g).mul_(hi - lo).add_(lo)

    def moments(self, *shape):
        """Activations: means of order one, variances well below."""
        return self.normal(*shape), self.uniform(*shape, lo=0.001, hi=0.2)

    def deltas(self, *shape):
        """What the output layer hands back: signed mean deltas, variance deltas that shrink the variance."""
        return self.normal(*shape, scale=0.1), self.uniform(*shape, lo=-0.2, hi=-0.001)

    def weights(self, fan_in, *shape):
        s = 1.0 / math.sqrt(fan_in)
        return self.normal(*shape, scale=s), self.uniform(*shape, lo=0.2 * s * s, hi=s * s)

    def relu_jcb(self, *shape):
        return (torch.rand(*shape, device="cuda", generator=self.g) < 0.6).float()


def _assign(g, tokens, experts, k, skew):
    """k different experts for every token, some experts liked more than others: the dispatch order (rows sorted by
    expert, tokens in order within one) and the offsets, on the device and as a list."""
    liking = g.normal(experts, scale=skew)
    noise = -torch.log(-torch.log(g.uniform(tokens, experts, lo=1e-6, hi=1.0 - 1e-6)))
    expert = torch.topk(liking + noise, k, dim=1).indices.reshape(-1)
    order = torch.argsort(expert, stable=True)
    token = (order // k).to(torch.int32)
    ends = torch.cumsum(torch.bincount(expert, minlength=experts), 0)
    offsets = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return token, offsets, offsets.tolist()


def _slots(g, tokens, k, idle):
    """Where each of a token's k slots lies in the dispatch order (-1: the slot has no expert), and how many do."""
    rank = torch.argsort(g.uniform(tokens * k))     # any order does: the rows are scattered as experts scatter them
    rank = rank[:int(tokens * k * (1.0 - idle))]
    pos = torch.full((tokens * k,), -1, dtype=torch.int32, device="cuda")
    pos[rank] = torch.arange(rank.numel(), dtype=torch.int32, device="cuda")
    return pos.reshape(tokens, k), rank.numel()


def _gates(g, pos):
    mu_g = g.uniform(*pos.shape, lo=0.05, hi=1.0)
    mu_g = mu_g * (pos >= 0)
    mu_g = mu_g / mu_g.sum(1, keepdim=True).clamp_min(1e-6)
    return mu_g, g.uniform(*pos.shape, lo=0.0, hi=0.05) * mu_g


def prepare(case, seed):
    c, g = case, _Gen(seed)
    s = dict(case)
    op = c["op"]
    if op in ("ln_fwd", "ln_bwd"):
        R, n = c["rows"], c["n"]
        s["mu_w"], s["var_w"] = 1.0 + g.normal(n, scale=0.1), g.uniform(n, lo=0.01, hi=0.2)
        s["mu_b"], s["var_b"] = g.normal(n, scale=0.1), g.uniform(n, lo=0.01, hi=0.2)
        s["mu_a"], s["var_a"] = g.moments(R, n)
        s["mu_a"] = s["mu_a"].mul_(g.uniform(R, 1, lo=0.3, hi=3.0)).add_(g.normal(R, 1))
        if not c["bias"]:
            s["mu_b"] = s["var_b"] = None
        if op == "ln_bwd":
            s["mu_row"] = s["mu_a"].mean(1)
            s["var_row"] = (s["mu_a"].var(1, unbiased=True) + s["var_a"].sum(1) / (n - 1)).contiguous()
            s["jcb"] = g.relu_jcb(R, n) if c["jcb"] else None
            s["dmu_o"], s["dvar_o"] = g.deltas(R, n)
    elif op == "route":
        T, E, k = c["tokens"], c["experts"], c["k"]
        s["mu_s"], s["var_s"] = g.normal(T, E) + g.normal(E, scale=0.5), g.uniform(T, E, lo=0.01, hi=0.5)
        if c["barred"]:
            bar = (g.uniform(T, E) < c["barred"]) | (g.uniform(T, 1) < 0.25 * c["barred"])
            s["mu_s"] = s["mu_s"].masked_fill_(bar, -math.inf)
        if c["train"]:
            s["dmu_g"], s["dvar_g"] = g.deltas(T, k)
    elif op.startswith("grouped"):
        T, E, k, K, N = c["tokens"], c["experts"], c["k"], c["K"], c["N"]
        s["token"], s["offsets"], s["ends"] = _assign(g, T, E, k, c["skew"])
        if op == "grouped_fwd":
            s["mu_w"], s["var_w"] = g.weights(K, E, N, K)
            s["mu_a"], s["var_a"] = g.moments(T, K)
        elif op == "grouped_state":
            s["mu_w"] = g.weights(K, E, N, K)[0]
            s["jcb"] = g.relu_jcb(T * k, K)
        else:
            s["var_w"] = g.weights(K, E, N, K)[1]
            s["mu_a"] = g.moments(T, K)[0]
        if op != "grouped_fwd":
            s["dmu_z"], s["dvar_z"] = g.deltas(T * k, N)
        if op != "grouped_state":
            s["mu_b"], s["var_b"] = g.weights(K, E, N) if c["bias"] else (None, None)
    else:
        T, k, N = c["tokens"], c["k"], c["N"]
        s["pos"], s["live"] = _slots(g, T, k, c["idle"])
        if op != "dispatch_bwd":
            s["mu_g"], s["var_g"] = _gates(g, s["pos"])
            s["mu_x"], s["var_x"] = g.moments(s["live"], N)
        if op == "combine_bwd":
            s["dmu_y"], s["dvar_y"] = g.deltas(T, N)
        if op == "dispatch_bwd":
            s["jcb"] = g.relu_jcb(T, N) if c["jcb"] else None
            s["dmu_x"], s["dvar_x"] = g.deltas(s["live"], N)
    return s


# --------------------------------------------------------------------------------------------------------- plain forms

def _ln_fwd(s):
    n = s["n"]
    mean = s["mu_a"].mean(1)
    d = s["mu_a"] - mean[:, None]
    var = ((d * d).sum(1) + s["var_a"].sum(1)) / (n - 1)
    inv = 1.0 / torch.sqrt(var + EPS)[:, None]
    w, vw = s["mu_w"], s["var_w"]
    mu_z = inv * d * w
    var_z = inv * inv * (s["var_a"] * (w * w + vw) + vw * d * d)
    if s["bias"]:
        mu_z, var_z = mu_z + s["mu_b"], var_z + s["var_b"]
    return dict(mu_row=mean, var_row=var, mu_z=mu_z, var_z=var_z)


def _ln_bwd(s):
    inv = 1.0 / torch.sqrt(s["var_row"] + EPS)[:, None]
    t = inv * s["mu_w"]
    if s["jcb"] is not None:
        t = t * s["jcb"]
    u = inv * (s["mu_a"] - s["mu_row"][:, None]) * s["var_w"]
    out = dict(dmu=t * s["dmu_o"], dvar=t * t * s["dvar_o"], dmu_w=(u * s["dmu_o"]).sum(0), dvar_w=(u * u * s["dvar_o"]).sum(0))
    if s["bias"]:
        out["dmu_b"] = s["var_b"] * s["dmu_o"].sum(0)
        out["dvar_b"] = s["var_b"] * s["var_b"] * s["dvar_o"].sum(0)
    return out


def _route(s):
    T, E, k = s["tokens"], s["experts"], s["k"]
    score, index = torch.sort(s["mu_s"].double(), dim=1, descending=True, stable=True)
    score, index = score[:, :k], index[:, :k]
    valid = score > -math.inf
    p = torch.where(valid, torch.exp(score - score[:, :1]), 0.0)
    g = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    v = torch.gather(s["var_s"].double(), 1, index)
    eye = torch.eye(k, dtype=torch.bool, device=g.device)
    # 1 - g_i as the sum of the others: it does not cancel where one gate is close to one
    rest = torch.where(eye, 0.0, g[:, None, :].expand(T, k, k)).sum(2)
    J = torch.where(eye, (g * rest)[:, :, None], -g[:, :, None] * g[:, None, :])
    var_g = (J * J * torch.where(valid, v, 0.0)[:, None, :]).sum(2)
    expert = torch.where(valid, index, E).reshape(-1)
    order = torch.argsort(expert, stable=True)
    ordered = expert[order]
    offsets = torch.searchsorted(ordered, torch.arange(E + 1, device=g.device))
    token = torch.where(ordered < E, order // k, -1)
    pos = torch.empty_like(order)
    pos[order] = torch.where(ordered < E, torch.arange(T * k, device=g.device), -1)
    i32 = torch.int32
    out = dict(expert=torch.where(valid, index, -1).to(i32), mu_g=g.float(), var_g=var_g.float(), offsets=offsets.to(i32),
               token=token.to(i32), pos=pos.to(i32).reshape(T, k))
    if s["train"]:
        dmu = (J * s["dmu_g"].double()[:, :, None]).sum(1)
        dvar = (J * J * s["dvar_g"].double()[:, :, None]).sum(1)
        out["dmu_s"] = torch.zeros_like(s["mu_s"]).scatter_(1, index, torch.where(valid, dmu, 0.0).float())
        out["dvar_s"] = torch.zeros_like(s["mu_s"]).scatter_(1, index, torch.where(valid, dvar, 0.0).float())
    return out


def _each(s):
    return [(e, slice(s["ends"][e], s["ends"][e + 1])) for e in range(s["experts"]) if s["ends"][e + 1] > s["ends"][e]]


def _grouped_fwd(s):
    a, v = s["mu_a"][s["token"]], s["var_a"][s["token"]]
    second = a * a + v
    def one(e, r):
        w, vw = s["mu_w"][e], s["var_w"][e]
        z, vz = a[r] @ w.t(), v[r] @ (w * w).t() + second[r] @ vw.t()
        return (z + s["mu_b"][e], vz + s["var_b"][e]) if s["bias"] else (z, vz)
    z, vz = zip(*[one(e, r) for e, r in _each(s)])
    return dict(mu_z=torch.cat(z), var_z=torch.cat(vz))


def _grouped_state(s):
    d = torch.cat([s["dmu_z"][r] @ s["mu_w"][e] for e, r in _each(s)])
    v = torch.cat([s["dvar_z"][r] @ (s["mu_w"][e] * s["mu_w"][e]) for e, r in _each(s)])
    return dict(dmu_a=s["jcb"] * d, dvar_a=s["jcb"] * s["jcb"] * v)


def _grouped_param(s):
    a = s["mu_a"][s["token"]]
    b = [slice(s["ends"][e], s["ends"][e + 1]) for e in range(s["experts"])]
    out = dict(dmu_w=s["var_w"] * torch.stack([s["dmu_z"][r].t() @ a[r] for r in b]),
               dvar_w=s["var_w"] * s["var_w"] * torch.stack([s["dvar_z"][r].t() @ (a[r] * a[r]) for r in b]))
    if s["bias"]:
        out["dmu_b"] = s["var_b"] * torch.stack([s["dmu_z"][r].sum(0) for r in b])
        out["dvar_b"] = s["var_b"] * s["var_b"] * torch.stack([s["dvar_z"][r].sum(0) for r in b])
    return out


def _taken(s, x):
    """[tokens, k, N]: the rows of the token's slots, zero where a slot has none."""
    pos = s["pos"].long()
    return torch.where((pos >= 0)[:, :, None], x[pos.clamp_min(0)], 0.0) if s["live"] else x.new_zeros(*pos.shape, s["N"])


def _combine_fwd(s):
    x, v = _taken(s, s["mu_x"]), _taken(s, s["var_x"])
    g, vg = s["mu_g"][:, :, None], s["var_g"][:, :, None]
    return dict(mu_y=(g * x).sum(1), var_y=(vg * (x * x + v) + g * g * v).sum(1))


def _combine_bwd(s):
    x = _taken(s, s["mu_x"])
    slot = s["pos"].reshape(-1)
    order = torch.argsort(slot)[slot.numel() - s["live"]:]      # the slots in the order of their rows
    g, t = s["mu_g"].reshape(-1)[order][:, None], order // s["k"]
    return dict(dmu_x=g * s["dmu_y"][t], dvar_x=g * g * s["dvar_y"][t], dmu_g=(x * s["dmu_y"][:, None, :]).sum(2),
                dvar_g=(x * x * s["dvar_y"][:, None, :]).sum(2))


def _dispatch_bwd(s):
    d, v = _taken(s, s["dmu_x"]).sum(1), _taken(s, s["dvar_x"]).sum(1)
    return dict(dmu_a=d, dvar_a=v) if s["jcb"] is None else dict(dmu_a=s["jcb"] * d, dvar_a=s["jcb"] * s["jcb"] * v)


PLAIN = dict(ln_fwd=_ln_fwd, ln_bwd=_ln_bwd, route=_route, grouped_fwd=_grouped_fwd, grouped_state=_grouped_state,
             grouped_param=_grouped_param, combine_fwd=_combine_fwd, combine_bwd=_combine_bwd, dispatch_bwd=_dispatch_bwd)


# ------------------------------------------------------------------------------------------------- the library's calls

def _call(s):
    from cutagi_b200 import ops
    op = s["op"]
    if op == "ln_fwd":
        z, vz, m, v = ops.layer_norm(s["mu_w"], s["var_w"], s["mu_b"], s["var_b"], s["mu_a"], s["var_a"], eps=EPS)
        return dict(mu_row=m, var_row=v, mu_z=z, var_z=vz)
    if op == "ln_bwd":
        names = ("dmu", "dvar", "dmu_w", "dvar_w") + (("dmu_b", "dvar_b") if s["bias"] else ())
        return dict(zip(names, ops.layer_norm_backward(s["mu_w"], s["var_w"], s["var_b"], s["mu_a"], s["jcb"], s["mu_row"],
                                                      s["var_row"], s["dmu_o"], s["dvar_o"], eps=EPS)))
    if op == "route":
        r = ops.route(s["mu_s"], s["var_s"], s["k"])
        out = dict(expert=r.expert, mu_g=r.mu_g, var_g=r.var_g, offsets=r.offsets, token=r.token, pos=r.pos)
        if s["train"]:
            out["dmu_s"], out["dvar_s"] = ops.route_backward(r, s["dmu_g"], s["dvar_g"])
        return out
    if op == "grouped_fwd":
        z, vz = ops.grouped_linear(s["mu_w"], s["var_w"], s["mu_b"], s["var_b"], s["mu_a"], s["var_a"], s["offsets"], s["token"])
        return dict(mu_z=z, var_z=vz)
    if op == "grouped_state":
        d, v = ops.grouped_linear_state(s["mu_w"], s["jcb"], s["dmu_z"], s["dvar_z"], s["offsets"])
        return dict(dmu_a=d, dvar_a=v)
    if op == "grouped_param":
        names = ("dmu_w", "dvar_w") + (("dmu_b", "dvar_b") if s["bias"] else ())
        return dict(zip(names, ops.grouped_linear_param(s["var_w"], s["var_b"], s["mu_a"], s["dmu_z"], s["dvar_z"],
                                                       s["offsets"], s["token"])))
    if op == "combine_fwd":
        y, vy = ops.combine(s["pos"], s["mu_g"], s["var_g"], s["mu_x"], s["var_x"])
        return dict(mu_y=y, var_y=vy)
    if op == "combine_bwd":
        return dict(zip(("dmu_x", "dvar_x", "dmu_g", "dvar_g"),
                        ops.combine_backward(s["pos"], s["mu_g"], s["mu_x"], None, s["dmu_y"], s["dvar_y"])))
    d, v = ops.dispatch_backward(s["pos"], s["jcb"], s["dmu_x"], s["dvar_x"])
    return dict(dmu_a=d, dvar_a=v)


def run(state):
    if own:
        return _call(state)
    return PLAIN[state["op"]](state)


# --------------------------------------------------------------------------------------------------------------- work

def work(case):
    c, op = case, case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        el, n, R = c["rows"] * c["n"], c["n"], c["rows"]
        if op == "ln_fwd":
            return dict(bytes=16 * el + 8 * R + (16 if c["bias"] else 8) * n, flops=14 * el)
        return dict(bytes=(24 if c["jcb"] else 20) * el + 8 * R + (28 if c["bias"] else 16) * n, flops=14 * el)
    if op == "route":
        T, E, k = c["tokens"], c["experts"], c["k"]
        # scores in; the chosen variances in; expert, two gate moments, token, pos out; deltas: two per slot in, two per score out
        b = 4 * T * E + 24 * T * k + 4 * (E + 1) + ((8 * T * k + 8 * T * E) if c["train"] else 0)
        return dict(bytes=b, flops=T * E + 6 * T * k * k)
    if op.startswith("grouped"):
        T, E, k, K, N = c["tokens"], c["experts"], c["k"], c["K"], c["N"]
        S, used = T * k, min(c["experts"], T * k)     # no more experts than rows can be asked for
        if op == "grouped_fwd":
            return dict(bytes=used * N * (8 * K + (8 if c["bias"] else 0)) + 8 * T * K + 8 * S * N + 4 * (S + E), flops=6 * S * K * N)
        if op == "grouped_state":
            return dict(bytes=4 * used * N * K + 8 * S * N + 12 * S * K + 4 * E, flops=4 * S * K * N)
        return dict(bytes=12 * E * N * K + (12 * E * N if c["bias"] else 0) + 4 * T * K + 8 * S * N + 4 * (S + E), flops=4 * S * K * N)
    T, k, N = c["tokens"], c["k"], c["N"]
    live = int(T * k * (1.0 - c["idle"]))
    if op == "combine_fwd":
        return dict(bytes=8 * live * N + 8 * T * N + 12 * T * k, flops=8 * live * N)
    if op == "combine_bwd":
        return dict(bytes=8 * T * N + 12 * live * N + 16 * T * k, flops=7 * live * N)
    return dict(bytes=8 * live * N + (12 if c["jcb"] else 8) * T * N + 4 * T * k, flops=2 * live * N)


# --------------------------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    f = {n: t.double() if torch.is_tensor(t) and t.dtype == torch.float32 else t for n, t in s.items()}
    if op == "ln_fwd":
        n = s["n"]
        mean = f["mu_a"].sum(1) / n
        # E[x^2] - mean^2 in 64 bits: the means here are of order one
        var = ((f["mu_a"] ** 2 + f["var_a"]).sum(1) - n * mean ** 2) / (n - 1)
        i2 = (1.0 / (var + EPS))[:, None]
        t2 = i2 * (f["mu_a"] - mean[:, None]) ** 2
        mu_z = torch.sign(f["mu_a"] - mean[:, None]) * torch.sqrt(t2) * f["mu_w"] + (f["mu_b"] if s["bias"] else 0.0)
        var_z = i2 * f["var_a"] * f["mu_w"] ** 2 + (i2 * f["var_a"] + t2) * f["var_w"] + (f["var_b"] if s["bias"] else 0.0)
        return dict(mu_row=mean, var_row=var, mu_z=mu_z, var_z=var_z)
    if op == "ln_bwd":
        i = (f["var_row"] + EPS) ** -0.5
        j = f["jcb"] if s["jcb"] is not None else torch.ones_like(f["mu_a"])
        hat = (f["mu_a"] - f["mu_row"][:, None]) * i[:, None]
        out = dict(dmu=torch.einsum("r,n,rn,rn->rn", i, f["mu_w"], j, f["dmu_o"]),
                   dvar=torch.einsum("r,n,rn,rn->rn", i * i, f["mu_w"] ** 2, j * j, f["dvar_o"]),
                   dmu_w=f["var_w"] * torch.einsum("rn,rn->n", hat, f["dmu_o"]),
                   dvar_w=f["var_w"] ** 2 * torch.einsum("rn,rn->n", hat * hat, f["dvar_o"]))
        if s["bias"]:
            out["dmu_b"], out["dvar_b"] = f["var_b"] * f["dmu_o"].sum(0), f["var_b"] ** 2 * f["dvar_o"].sum(0)
        return out
    if op == "route":
        return _exact_route(s)
    if op.startswith("grouped"):
        return _exact_grouped(s, f)
    return _exact_rows(s, f)


def _exact_route(s):
    T, E, k = s["tokens"], s["experts"], s["k"]
    mu, var = s["mu_s"].cpu().numpy().astype(np.float64), s["var_s"].cpu().numpy().astype(np.float64)
    idx = np.argsort(-mu, axis=1, kind="stable")[:, :k]
    sel, v = np.take_along_axis(mu, idx, 1), np.take_along_axis(var, idx, 1)
    ok = np.isfinite(sel)
    top = np.where(ok[:, :1], sel[:, :1], 0.0)
    p = np.where(ok, np.exp(np.where(ok, sel - top, 0.0)), 0.0)
    z = np.maximum(p.sum(1, keepdims=True), 1e-300)
    g = p / z
    others = p[:, None, :] * (1.0 - np.eye(k))[None]            # weights of the other chosen experts
    rest = others.sum(2) / z
    v = np.where(ok, v, 0.0)
    var_g = g * g * (rest * rest * v + ((others / z[:, :, None]) ** 2 * v[:, None, :]).sum(2))
    out = dict(expert=None, mu_g=g, var_g=var_g, offsets=None, token=None, pos=None)
    if s["train"]:
        d, w = s["dmu_g"].cpu().numpy().astype(np.float64), s["dvar_g"].cpu().numpy().astype(np.float64)
        dmu = g * (rest * d - (others / z[:, :, None] * d[:, None, :]).sum(2))
        dvar = g * g * (rest * rest * w + ((others / z[:, :, None]) ** 2 * w[:, None, :]).sum(2))
        for name, val in (("dmu_s", dmu), ("dvar_s", dvar)):
            full = np.zeros((T, E))
            np.put_along_axis(full, idx, np.where(ok, val, 0.0), 1)
            out[name] = full
    return out


def _exact_grouped(s, f):
    op, ends = s["op"], s["ends"]
    if 6.0 * s["tokens"] * s["k"] * s["K"] * s["N"] > 4e12:
        return None
    parts = []
    for e in range(s["experts"]):
        r = slice(ends[e], ends[e + 1])
        t = s["token"][r].long()
        if op == "grouped_fwd":
            w, a, v = f["mu_w"][e], f["mu_a"][t], f["var_a"][t]
            z = torch.einsum("bk,nk->bn", a, w)
            vz = torch.einsum("bk,nk->bn", v, w * w + f["var_w"][e]) + torch.einsum("bk,nk->bn", a * a, f["var_w"][e])
            parts.append((z + f["mu_b"][e], vz + f["var_b"][e]) if s["bias"] else (z, vz))
        elif op == "grouped_state":
            w, j = f["mu_w"][e], f["jcb"][r]
            parts.append((torch.einsum("bn,nk->bk", f["dmu_z"][r], w) * j, torch.einsum("bn,nk->bk", f["dvar_z"][r], w * w) * j * j))
        else:
            a, d, v, vw = f["mu_a"][t], f["dmu_z"][r], f["dvar_z"][r], f["var_w"][e]
            got = [vw * torch.einsum("bn,bk->nk", d, a), vw * vw * torch.einsum("bn,bk->nk", v, a * a)]
            if s["bias"]:
                got += [f["var_b"][e] * d.sum(0), f["var_b"][e] ** 2 * v.sum(0)]
            parts.append(got)
    join = torch.stack if op == "grouped_param" else torch.cat
    names = {"grouped_fwd": ("mu_z", "var_z"), "grouped_state": ("dmu_a", "dvar_a"),
             "grouped_param": ("dmu_w", "dvar_w", "dmu_b", "dvar_b")}[op]
    return {n: join([p[i] for p in parts]) for i, n in enumerate(names[:len(parts[0])])}


def _exact_rows(s, f):
    T, k, N, live = s["tokens"], s["k"], s["N"], s["live"]
    row = s["pos"].reshape(-1).long()
    slot = torch.nonzero(row >= 0).reshape(-1)
    row, tok = row[slot], slot // k
    if s["op"] == "combine_bwd":
        dx, vx = torch.empty(live, N, dtype=torch.float64, device="cuda"), torch.empty(live, N, dtype=torch.float64, device="cuda")
        g = f["mu_g"].reshape(-1)[slot][:, None]
        dx[row], vx[row] = g * f["dmu_y"][tok], g * g * f["dvar_y"][tok]
        dg, vg = torch.zeros(T * k, dtype=torch.float64, device="cuda"), torch.zeros(T * k, dtype=torch.float64, device="cuda")
        dg[slot] = torch.einsum("sn,sn->s", f["mu_x"][row], f["dmu_y"][tok])
        vg[slot] = torch.einsum("sn,sn->s", f["mu_x"][row] ** 2, f["dvar_y"][tok])
        return dict(dmu_x=dx, dvar_x=vx, dmu_g=dg.reshape(T, k), dvar_g=vg.reshape(T, k))
    y, vy = torch.zeros(T, N, dtype=torch.float64, device="cuda"), torch.zeros(T, N, dtype=torch.float64, device="cuda")
    if s["op"] == "combine_fwd":
        g, vg = f["mu_g"].reshape(-1)[slot][:, None], f["var_g"].reshape(-1)[slot][:, None]
        x, v = f["mu_x"][row], f["var_x"][row]
        y.index_add_(0, tok, g * x)
        vy.index_add_(0, tok, (vg + g * g) * v + vg * x * x)
        return dict(mu_y=y, var_y=vy)
    y.index_add_(0, tok, f["dmu_x"][row])
    vy.index_add_(0, tok, f["dvar_x"][row])
    return dict(dmu_a=y, dvar_a=vy) if s["jcb"] is None else dict(dmu_a=y * f["jcb"], dvar_a=vy * f["jcb"] ** 2)
