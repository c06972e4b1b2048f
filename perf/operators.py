"""Workloads of the sequence and expert operators: the gated linear recurrence
with its gradient, and the matrix products grouped by expert with theirs.

Where `own` is false, `run` computes them from elementary torch operations in
64 bits (DS results carry about 48 bits, more than 32-bit sums keep); where
it is true, it makes the calls a user makes of `ds_b200.ops`.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"f64": torch.float64, "f32": torch.float32}


def listed():
    def rec(name, op, type, B, T, D, resets=0):
        # resets: a document starts (a_t = 0) every so many steps on average
        return {"name": name, "op": op, "type": type, "B": B, "T": T, "D": D, "resets": resets}

    def dot(name, op, M, K, N, G, skew, tail):
        # skew: spread of the experts' popularity; tail: rows behind the last group
        return {"name": name, "op": op, "type": "f64", "M": M, "K": K, "N": N, "G": G,
                "skew": skew, "tail": tail}

    return [
        # serving: the state of 64 sequences advanced by one token
        rec("recurrence, one token", "recurrence", "f64", 64, 1, 4096),
        # a training batch of a recurrent layer
        rec("recurrence, batch", "recurrence", "f64", 8, 2048, 1024),
        # prefill of one long sequence, few channels and an odd number of them
        rec("recurrence, long", "recurrence", "f64", 1, 65536, 250),
        # packed documents in f32: the gate is zero where a document starts
        rec("recurrence, documents", "recurrence", "f32", 4, 4096, 2048, 700),
        # the training batch's gradient
        rec("recurrence gradient, batch", "recurrence_vjp", "f64", 8, 2048, 1024),
        # odd sizes in f32
        rec("recurrence gradient, odd", "recurrence_vjp", "f32", 3, 1337, 517, 300),
        # serving: a few tokens, each at its own expert
        dot("experts, decode", "ragged_dot", 16, 1024, 2048, 16, 1.0, 0),
        # odd sizes, some experts without tokens, padding behind the last group
        dot("experts, odd", "ragged_dot", 1500, 777, 1001, 13, 2.0, 37),
        # a training batch's products, experts of unequal popularity
        dot("experts, batch", "ragged_dot", 8192, 2048, 2048, 8, 0.7, 0),
        # the gradient of its tokens: the experts' matrices transposed
        dot("experts, token gradient", "ragged_dot_t", 8192, 2048, 2048, 8, 0.7, 0),
        # the gradient of its experts' matrices
        dot("experts, matrix gradient", "ragged_dot_contract", 8192, 2048, 2048, 8, 0.7, 0),
        # the same with many experts, few tokens each
        dot("experts, matrix gradient odd", "ragged_dot_contract", 1111, 300, 515, 20, 1.5, 50),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence_vjp", "ragged_dot", "ragged_dot_t",
                     "ragged_dot_contract"])
    if op.startswith("recurrence"):
        D = _log(rng, 1, 4096)
        # at most the batch's 2^24 values
        T = _log(rng, 1, min(65536, max(1, (1 << 24) // D)))
        B = _log(rng, 1, min(64, max(1, (1 << 24) // (D * T))))
        return {"op": op, "type": rng.choice(["f64", "f32"]), "B": B, "T": T, "D": D,
                "resets": rng.choice([0, 0, 50, 1000])}
    K, N = _log(rng, 16, 2048), _log(rng, 16, 2048)
    M = _log(rng, 1, 8192)
    G = _log(rng, 1, 64)
    while G * K * N > 8 * 2048 * 2048:
        G = max(1, G // 2)
    return {"op": op, "type": "f64", "M": M, "K": K, "N": N, "G": G,
            "skew": rng.uniform(0.0, 2.5), "tail": rng.choice([0, 0, rng.randint(0, M // 4)])}


def _sizes(case, seed):
    """Rows per group: every row but the tail's takes an expert at random,
    experts differing in popularity by a log-normal factor."""
    r = np.random.default_rng([seed, 7])
    p = np.exp(case["skew"] * r.standard_normal(case["G"]))
    return r.multinomial(case["M"] - case["tail"], p / p.sum()).tolist()


def _inputs(case, seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, dtype=torch.float64, device=device)

    def uniform(*shape):
        return torch.rand(shape, generator=g, dtype=torch.float64, device=device)

    if case["op"].startswith("recurrence"):
        t = _TYPES[case["type"]]
        B, T, D = case["B"], case["T"], case["D"]
        # gates sigmoid(2 + x), most near one, as a trained layer has them
        a = torch.sigmoid(2.0 + 1.5 * normal(B, T, D))
        if case["resets"]:
            a = a * (uniform(B, T, 1) * case["resets"] >= 1.0)
        s = {"a": a.to(t), "h0": normal(B, D).to(t)}
        if case["op"] == "recurrence":
            s["b"] = normal(B, T, D).to(t)
        else:
            s["h"] = (2.0 * normal(B, T, D)).to(t)
            s["grad"] = normal(B, T, D).to(t)
        return s
    M, K, N, G = case["M"], case["K"], case["N"], case["G"]
    sizes = _sizes(case, seed)
    s = {"sizes": sizes, "group_sizes": torch.tensor(sizes, dtype=torch.int32, device=device)}
    if case["op"] == "ragged_dot":
        s["lhs"], s["rhs"] = normal(M, K), normal(G, K, N) / math.sqrt(K)
    elif case["op"] == "ragged_dot_t":
        s["lhs"], s["rhs"] = normal(M, K), normal(G, N, K) / math.sqrt(K)
    else:
        s["lhs"], s["rhs"] = normal(M, K), normal(M, N)
    return s


def prepare(case, seed):
    s = _inputs(case, seed, torch.device("cuda"))
    s["op"], s["type"] = case["op"], case["type"]
    return s


# ---- plain forms ----------------------------------------------------------------

def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t (h_{-1} = 0) along dim 1, by doubling the span
    each position has taken in."""
    T, d = a.shape[1], 1
    while d < T:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], dim=1)
        if 2 * d < T:
            a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], dim=1)
        d *= 2
    return b


def _recurrence(a, b, h0):
    t = a.dtype
    a, b, h0 = a.double(), b.double(), h0.double()
    b = torch.cat([b[:, :1] + a[:, :1] * h0.unsqueeze(1), b[:, 1:]], dim=1)
    return _scan(a, b).to(t)


def _recurrence_vjp(a, h, grad, h0):
    t = a.dtype
    a, h, grad, h0 = a.double(), h.double(), grad.double(), h0.double()
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    db = _scan(after.flip(1), grad.flip(1)).flip(1)
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], dim=1)
    return (db * before).to(t), db.to(t), (a[:, 0] * db[:, 0]).to(t)


def _groups(x, sizes):
    return x[:sum(sizes)].split(sizes)


def _ragged_dot(lhs, rhs, sizes):
    rows = [x @ w for x, w in zip(_groups(lhs, sizes), rhs)]
    return torch.cat(rows + [lhs.new_zeros(lhs.shape[0] - sum(sizes), rhs.shape[-1])])


def _ragged_dot_contract(lhs, rhs, sizes):
    return torch.stack([x.T @ y for x, y in zip(_groups(lhs, sizes), _groups(rhs, sizes))])


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "ds-experiment_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ds_b200 import ops
    return ops


def run(state):
    op = state["op"]
    if own:
        ops = _ops()
        t = state["type"]
        if op == "recurrence":
            call = ops.ds_linear_recurrence_f64 if t == "f64" else ops.ds_linear_recurrence_f32
            return call(state["a"], state["b"], state["h0"])
        if op == "recurrence_vjp":
            call = (ops.ds_linear_recurrence_vjp_f64 if t == "f64"
                    else ops.ds_linear_recurrence_vjp_f32)
            return call(state["a"], state["h"], state["grad"], state["h0"])
        if op == "ragged_dot":
            return ops.ds_ragged_dot_f64(state["lhs"], state["rhs"], state["group_sizes"])
        if op == "ragged_dot_t":
            return ops.ds_ragged_dot_f64(state["lhs"], state["rhs"], state["group_sizes"],
                                         rhs_contracting=2)
        return ops.ds_ragged_dot_contract_f64(state["lhs"], state["rhs"], state["group_sizes"])
    if op == "recurrence":
        return _recurrence(state["a"], state["b"], state["h0"])
    if op == "recurrence_vjp":
        return _recurrence_vjp(state["a"], state["h"], state["grad"], state["h0"])
    if op == "ragged_dot":
        return _ragged_dot(state["lhs"], state["rhs"], state["sizes"])
    if op == "ragged_dot_t":
        return _ragged_dot(state["lhs"], state["rhs"].transpose(1, 2), state["sizes"])
    return _ragged_dot_contract(state["lhs"], state["rhs"], state["sizes"])


def work(case):
    if case["op"].startswith("recurrence"):
        n, state = case["B"] * case["T"] * case["D"], case["B"] * case["D"]
        e = 8 if case["type"] == "f64" else 4
        if case["op"] == "recurrence":
            return {"bytes": e * (3 * n + state), "flops": 2 * n}
        return {"bytes": e * (5 * n + 2 * state), "flops": 3 * n}
    M, K, N, G = case["M"], case["K"], case["N"], case["G"]
    rows = M - case["tail"]
    if case["op"] == "ragged_dot_contract":
        return {"bytes": 8 * (rows * (K + N) + G * K * N) + 4 * G, "flops": 2 * rows * K * N}
    # a group without rows need not read its matrix: the groups that have some
    # when every row takes one at random
    used = G * (1.0 - (1.0 - 1.0 / G) ** rows)
    return {"bytes": int(8 * (rows * K + M * N + used * K * N)) + 4 * G,
            "flops": 2 * rows * K * N}


# ---- the definition in 64 bits, step by step on the host ---------------------------

def exact(case, seed):
    s = _inputs(case, seed, torch.device("cuda"))
    x = {k: v.double().cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "recurrence":
        a, b, h = x["a"], x["b"], x["h0"]
        out = np.empty_like(b)
        for t in range(b.shape[1]):
            h = a[:, t] * h + b[:, t]
            out[:, t] = h
        return torch.from_numpy(out)
    if case["op"] == "recurrence_vjp":
        a, h, grad, h0 = x["a"], x["h"], x["grad"], x["h0"]
        da, db = np.empty_like(a), np.empty_like(a)
        g = np.zeros_like(h0)
        for t in reversed(range(a.shape[1])):
            g = g + grad[:, t]
            db[:, t] = g
            da[:, t] = g * (h[:, t - 1] if t else h0)
            g = a[:, t] * g
        return torch.from_numpy(da), torch.from_numpy(db), torch.from_numpy(g)
    lhs, rhs = x["lhs"], x["rhs"]
    ends = np.cumsum(s["sizes"])
    if case["op"] == "ragged_dot_contract":
        out = np.zeros((case["G"], case["K"], case["N"]))
        for g, (n, e) in enumerate(zip(s["sizes"], ends)):
            out[g] = np.matmul(lhs[e - n:e].T, rhs[e - n:e])
        return torch.from_numpy(out)
    out = np.zeros((case["M"], case["N"]))
    for g, (n, e) in enumerate(zip(s["sizes"], ends)):
        w = rhs[g] if case["op"] == "ragged_dot" else rhs[g].T
        out[e - n:e] = np.matmul(lhs[e - n:e], w)
    return torch.from_numpy(out)
