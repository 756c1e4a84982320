"""Cases that measure two operators of a language model's training step: the softmax cross entropy of a
linear output layer over a large vocabulary, whose scores are never kept, with its gradients; and the
global norm of all gradients with the clipping by it, as the update applies it.

`run` computes each in its plain form (elementary torch operations on the whole score matrix, on one
flat gradient buffer), or through the package's public functions when `own` is set.  Arrays are
column-major as the package holds them: a (V, H) weight matrix is a flat tensor whose rows are
contiguous along V, its transposed form (H, V) one that is contiguous along H.  Labels are 1-based, 0
leaves an instance out."""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The head's work is V*H*N; no drawn case exceeds these (the largest listed one's).
MOST_PRODUCT = 50257 * 1024 * 4096
MOST_WEIGHTS = 32000 * 4096
MOST_SCORES = 50257 * 4096
MOST_PARAMS = 24 * (4096 * 4096 + 4096)


def _package():
    path = os.path.join(ROOT, "knet.jl_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import knet_sm100
    return knet_sm100


def _head(name, V, H, N, trans, back, bias, skip, bits=32):
    return {"name": name, "op": "head", "V": V, "H": H, "N": N, "trans": trans, "back": back, "bias": bias, "skip": skip, "bits": bits}


def _clip(name, opt, arrays, total, bits=32, scale=1.0, above=True):
    return {"name": name, "op": "clip", "opt": opt, "arrays": arrays, "total": total, "bits": bits, "scale": scale, "above": above}


def listed():
    return [
        # the tutorial's classifier on a batch of 100: launches are all that counts
        _head("head 10x64 n100", 10, 64, 100, False, True, True, 0.0),
        # the score of one token under an embedding that is also the output matrix
        _head("score 50257x1024 n1", 50257, 1024, 1, True, False, False, 0.0),
        # scoring a validation batch
        _head("score 50257x1024 n2048", 50257, 1024, 2048, False, False, True, 0.0),
        # one training step of that model; a padded batch leaves some positions out
        _head("train 50257x1024 n4096 tied", 50257, 1024, 4096, True, True, False, 0.0625),
        # a wide model with few tokens per step: the weights outweigh the instances
        _head("train 32000x4096 n512", 32000, 4096, 512, False, True, False, 0.0),
        # the output layer of the data-parallel MLP: many instances, few classes
        _head("train 1000x8192 n8192", 1000, 8192, 8192, False, True, True, 0.0),
        # sizes that divide nothing
        _head("train 10007x515 n333", 10007, 515, 333, False, True, True, 0.125),
        # the same operator on Float64 arrays
        _head("train 1000x784 n512 f64", 1000, 784, 512, False, True, True, 0.0, 64),
        # the parameters of the 784-64-10 tutorial model: launches again
        _clip("clip adam 4 arrays", "adam", 4, 784 * 64 + 64 + 64 * 10 + 10),
        # 24 matrices of 4096x4096 and 24 bias vectors
        _clip("clip adam 48 arrays", "adam", 48, MOST_PARAMS),
        # a model of many small and some large arrays, gradients summed over 8 ranks
        _clip("clip momentum 301 arrays", "momentum", 301, 30_000_019, scale=0.125),
        # gradients clipped in place for an optimizer that updates array by array
        _clip("clip in place f64", "inplace", 37, 9_000_001, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        bits = 64 if rng.random() < 0.15 else 32
        shrink = 16 if bits == 64 else 1        # Float64 products run at a fraction of the rate
        V, H = _log(rng, 10, 50257), _log(rng, 64, 8192)
        H = min(H, MOST_WEIGHTS // V)
        N = min(_log(rng, 1, 8192), MOST_SCORES // V, max(1, MOST_PRODUCT // shrink // (V * H)))
        return {"op": "head", "V": V, "H": H, "N": N, "trans": rng.random() < 0.5, "back": rng.random() < 0.7,
                "bias": rng.random() < 0.5, "skip": rng.choice([0.0, 0.03, 0.2]), "bits": bits}
    opt = rng.choice(["adam", "adam", "momentum", "sgd", "inplace"])
    bits = 64 if rng.random() < 0.2 else 32
    arrays = _log(rng, 1, 400)
    total = max(_log(rng, 10_000, MOST_PARAMS // (2 if bits == 64 else 1)), 16 * arrays)
    return {"op": "clip", "opt": opt, "arrays": arrays, "total": total, "bits": bits,
            "scale": rng.choice([1.0, 0.5, 0.125]), "above": rng.random() < 0.8}


def _sizes(case):
    """How the flat buffer is cut into arrays: 24 equal layers of a matrix and a bias for the 48, else matrices
    and vectors whose sizes spread over their logarithm."""
    n, total = case["arrays"], case["total"]
    if n == 48 and total == MOST_PARAMS:
        return [4096 * 4096, 4096] * 24
    if n == 4 and total == 784 * 64 + 64 + 64 * 10 + 10:
        return [784 * 64, 64, 64 * 10, 10]
    rng = random.Random(1000 * n + total)
    parts = [math.exp(rng.uniform(0, 9)) for _ in range(n)]
    rest = total - n
    sizes = [1 + int(rest * p / sum(parts)) for p in parts]
    sizes[0] += total - sum(sizes)
    return sizes


def _dtype(case):
    return torch.float64 if case["bits"] == 64 else torch.float32


# ---- inputs -----------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 13)
    dt = _dtype(case)

    def normal(n, std):
        return torch.randn(n, generator=g, device="cuda", dtype=dt).mul_(std)

    if case["op"] == "head":
        V, H, N = case["V"], case["H"], case["N"]
        s = {"case": case, "w": normal(V * H, 3.0 / math.sqrt(H)), "x": normal(H * N, 1.0)}      # scores of about N(0, 3)
        s["b"] = normal(V, 0.5) if case["bias"] else None
        lab = torch.randint(1, V + 1, (N,), generator=g, device="cuda", dtype=torch.int32)
        gone = torch.rand(N, generator=g, device="cuda") < case["skip"]
        gone[0] = False
        s["labels"] = torch.where(gone, torch.zeros_like(lab), lab)
        if own:
            K = _package()
            s["K"] = K
            s["kw"] = K.KnetArray(s["w"], (H, V) if case["trans"] else (V, H))
            s["kx"] = K.KnetArray(s["x"], (H, N))
            s["kb"] = None if s["b"] is None else K.KnetArray(s["b"], (V,))
        return s
    n = case["total"]
    s = {"case": case, "t": 0, "g": normal(n, 1e-3)}
    # the norm of gscale*g is close to 1e-3*scale*sqrt(n)
    s["limit"] = 1e-3 * case["scale"] * math.sqrt(n) * (0.5 if case["above"] else 2.0)
    if case["opt"] == "inplace":
        s["fresh"] = s["g"].clone()
    else:
        s["w"] = normal(n, 0.02)
        s["m"] = torch.zeros_like(s["g"]) if case["opt"] != "sgd" else None
        s["v"] = torch.zeros_like(s["g"]) if case["opt"] == "adam" else None
    if own:
        K = _package()
        s["K"] = K
        arrays, at = [], 0
        flat = [a for a in (s.get("w", s["g"]), s["g"], s.get("m"), s.get("v")) if a is not None]
        for size in _sizes(case):
            arrays.append(tuple(a[at:at + size] for a in flat))
            at += size
        s["plan"] = K.MultiTensorPlan(arrays)
        s["rule"] = {"adam": K.Adam(), "momentum": K.Momentum(lr=0.05, gamma=0.9), "sgd": K.SGD(lr=0.1), "inplace": None}[case["opt"]]
    return s


# ---- one pass ---------------------------------------------------------------------------------------
def run(s):
    if s["case"]["op"] == "head":
        return _head_own(s) if own else _head_plain(s)
    return _clip_own(s) if own else _clip_plain(s)


def _head_own(s):
    K, case = s["K"], s["case"]
    res = K.ops.linear_nll_device(s["kw"], s["kx"], s["labels"], b=s["kb"], trans=case["trans"])
    out = {"total": res.total, "count": res.count, "lse": res.lse}
    if case["back"]:
        dw, dx, db = K.ops.linear_nll_back(s["kw"], s["kx"], res, b=s["kb"], trans=case["trans"])
        out["dw"], out["dx"] = dw.data, dx.data
        if db is not None:
            out["db"] = db.data
    return out


def _head_plain(s):
    case = s["case"]
    V, H, N = case["V"], case["H"], case["N"]
    x = s["x"].view(N, H)
    w = s["w"].view(V, H).t() if case["trans"] else s["w"].view(H, V)           # (H, V)
    scores = x @ w
    if s["b"] is not None:
        scores = scores + s["b"]
    used = s["labels"] != 0
    at = (s["labels"].long() - 1).clamp_min(0).unsqueeze(1)
    top = scores.max(1, keepdim=True).values
    e = torch.exp(scores - top)
    z = e.sum(1, keepdim=True)
    lse = (top + torch.log(z)).squeeze(1)
    per = torch.where(used, lse - scores.gather(1, at).squeeze(1), torch.zeros_like(lse))
    count = used.sum().to(torch.int32).view(1)
    out = {"total": per.sum().view(1), "count": count, "lse": lse}
    if case["back"]:
        ds = e / z
        ds.scatter_add_(1, at, torch.full_like(z, -1.0))
        ds = ds * (used.to(ds.dtype) / count).unsqueeze(1)
        out["dx"] = (ds @ w.t()).reshape(-1)
        out["dw"] = (ds.t() @ x if case["trans"] else x.t() @ ds).reshape(-1)
        if s["b"] is not None:
            out["db"] = ds.sum(0)
    return out


def _clip_own(s):
    K, case = s["K"], s["case"]
    if case["opt"] == "inplace":
        s["g"].copy_(s["fresh"])                       # what a backward pass leaves
        norm = K.train.gclip_global_(s["plan"], s["limit"], gscale=case["scale"])
        return {"norm": norm, "g": s["g"]}
    norm = K.update_multi_(s["plan"], s["rule"], case["scale"], gclip_global=s["limit"])
    return {"norm": norm, **{k: s[k] for k in ("w", "m", "v") if s[k] is not None}}


def _clip_plain(s):
    case = s["case"]
    if case["opt"] == "inplace":
        s["g"].copy_(s["fresh"])
    norm = s["g"].double().square().sum().sqrt().view(1) * case["scale"]
    factor = torch.where(norm > s["limit"], s["limit"] / norm, torch.ones_like(norm)).to(s["g"].dtype)
    if case["opt"] == "inplace":
        s["g"].mul_(factor)
        return {"norm": norm, "g": s["g"]}
    g = s["g"] * case["scale"] * factor
    w, m, v = s["w"], s["m"], s["v"]
    s["t"] += 1
    if case["opt"] == "sgd":
        w.sub_(g * 0.1)
    elif case["opt"] == "momentum":
        m.mul_(0.9).sub_(g * 0.05)
        w.add_(m)
    else:
        m.mul_(0.9).add_(g * 0.1)
        v.mul_(0.999).add_(g * g * 0.001)
        w.sub_(0.001 * (m / (1 - 0.9 ** s["t"])) / (torch.sqrt(v / (1 - 0.999 ** s["t"])) + 1e-8))
    return {"norm": norm, **{k: s[k] for k in ("w", "m", "v") if s[k] is not None}}


# ---- what a pass cannot do without ------------------------------------------------------------------
def work(case):
    size = case["bits"] // 8
    if case["op"] == "head":
        V, H, N = case["V"], case["H"], case["N"]
        vec = V if case["bias"] else 0
        values, flops = V * H + H * N + vec + N, 2.0 * V * H * N
        if case["back"]:                       # the scores once more, dx and dw; w and x again, dw, dx and db written
            values += 2 * V * H + 2 * H * N + 2 * vec
            flops += 6.0 * V * H * N
        return {"bytes": size * values + 4 * N, "flops": flops}
    n = case["total"]
    # the norm reads g; then update! reads w, g and its state and writes w and the state; in place reads and writes g
    # (and the pass begins with a copy of fresh gradients)
    values = {"adam": 8, "momentum": 6, "sgd": 4, "inplace": 5 if case["above"] else 3}[case["opt"]]
    return {"bytes": size * n * values, "flops": 2.0 * n + {"adam": 14, "momentum": 4, "sgd": 2, "inplace": 1}[case["opt"]] * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    global own
    kept, own = own, False
    s = prepare(case, seed)
    own = kept
    if case["op"] == "head":
        return _head_exact(case, s)
    g = s["g"].to(torch.float64) * case["scale"]
    norm = torch.linalg.vector_norm(g).reshape(1)
    if float(norm) > s["limit"]:
        g = g * (s["limit"] / norm)
    if case["opt"] == "inplace":
        return {"norm": norm, "g": g / case["scale"]}
    w = s["w"].to(torch.float64)
    if case["opt"] == "sgd":
        return {"norm": norm, "w": w - 0.1 * g}
    if case["opt"] == "momentum":
        return {"norm": norm, "w": w - 0.05 * g, "m": -0.05 * g}
    # the first step of Adam from zero moments: the bias-corrected moments are g and g^2
    return {"norm": norm, "w": w - 0.001 * g / (g.abs() + 1e-8), "m": 0.1 * g, "v": 0.001 * g.square()}


def _head_exact(case, s):
    V, H, N = case["V"], case["H"], case["N"]
    x = s["x"].to(torch.float64).reshape(N, H)
    w = s["w"].to(torch.float64)
    w = w.reshape(V, H) if case["trans"] else w.reshape(H, V).t()
    scores = torch.mm(w, x.t())                                                 # (V, N)
    if s["b"] is not None:
        scores += s["b"].to(torch.float64)[:, None]
    lse = torch.logsumexp(scores, 0)
    inst = torch.nonzero(s["labels"] != 0).squeeze(1)
    rows = s["labels"][inst].long() - 1
    out = {"total": (lse[inst] - scores[rows, inst]).sum().reshape(1), "count": None, "lse": lse}
    if case["back"]:
        p = torch.zeros_like(scores)
        p[:, inst] = torch.exp(scores[:, inst] - lse[inst])
        p[rows, inst] -= 1.0
        p /= inst.numel()
        out["dx"] = torch.mm(p.t(), w).reshape(-1)
        dw = torch.mm(p, x)
        out["dw"] = (dw if case["trans"] else dw.t()).reshape(-1)
        if s["b"] is not None:
            out["db"] = p.sum(1)
    return out
