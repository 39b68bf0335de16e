"""Cases and plain forms of the operators a training generation is made of: choosing moves from scores (sample_actions), the
normalisation layer of a residual tower with its gradient (group_norm_act) and the orthogonalised weight update (orthogonalize).

``run`` computes a case in elementary torch operations, or, where ``own`` is true, through alphazero_amd.ops."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
GN_EPS = 1e-5


# ------------------------------------------------------------------------------------------------ cases
def _sampling(name, rows, n, dtype, temperature, top_k, top_p, min_p, legal, spread):
    """temperature: one number, or "rows": another one per row.  legal: a mask of legal moves comes along.
    spread: standard deviation of the scores"""
    return {"name": name, "op": "sample", "rows": rows, "n": n, "dtype": dtype, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "legal": legal, "spread": spread}


def _norm(name, n, c, h, w, groups, dtype, act, residual, train):
    return {"name": name, "op": "norm", "n": n, "c": c, "h": h, "w": w, "groups": groups, "dtype": dtype, "act": act,
            "residual": residual, "train": train}


def _ortho(name, shapes, dtype):
    """shapes: "rows x cols x how many" terms joined by spaces"""
    return {"name": name, "op": "ortho", "shapes": shapes, "dtype": dtype}


def listed():
    return [
        # one game's move on the 15x15 board: the call is latency
        _sampling("sample_one_game", 1, 225, "f32", 1.0, 0, 0.95, 0.0, True, 2.0),
        # the opening moves of 16,384 games at once, every game with its own temperature
        _sampling("sample_all_games", 16384, 225, "f32", "rows", 16, 0.9, 0.02, True, 2.0),
        # one long row: few rows, much to read
        _sampling("sample_one_long_row", 1, 131072, "bf16", 0.8, 50, 0.95, 0.0, False, 3.0),
        # a large batch of long rows of an odd length
        _sampling("sample_long_rows", 512, 65537, "bf16", 0.7, 0, 0.9, 0.001, False, 3.0),
        # a training batch of the default size on the 9x9 board: launches count
        _norm("norm_train_small", 64, 64, 9, 9, 8, "f32", "relu", False, True),
        # the tail of a residual block in the learner: 128 channels on the 15x15 board, batch 1,024, float32
        _norm("norm_train_block", 1024, 128, 15, 15, 8, "f32", "relu", True, True),
        # the self-play batch in bf16, no gradients
        _norm("norm_play", 16384, 64, 15, 15, 8, "bf16", "relu", False, False),
        # few samples with large planes of an odd width: a sample does not fit one workgroup
        _norm("norm_train_planes", 4, 512, 128, 127, 32, "f16", "silu", False, True),
        # one 3x3 convolution's update
        _ortho("ortho_one_conv", "64x576x1", "f32"),
        # every matrix of the deep 128-channel net: 20 convolutions, the stem, the policy and value layers
        _ortho("ortho_deep_net", "128x1152x20 128x81x1 225x225x1 64x450x1", "f32"),
        # a tall odd-sized float32 matrix
        _ortho("ortho_tall", "2501x1203x1", "f32"),
        # a large square matrix in bf16: the matrix rate counts
        _ortho("ortho_large", "4096x4096x1", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(["sample", "norm", "ortho"])
    if op == "sample":
        n = _log_int(rng, 9, 131072)  # from the 9 actions of tic-tac-toe on
        rows = _log_int(rng, 1 if n > 200 else 32, min(16384, max(1, 512 * 65537 // n)))
        case = _sampling("", rows, n, rng.choice(list(DTYPES)), rng.choice(["rows", 1.0, 0.5, 0.1, 1.5, 0.0]),
                         rng.choice([0, 0, 1, _log_int(rng, 1, n + 5)]), rng.choice([1.0, 0.95, 0.9, 0.5, 0.1]),
                         rng.choice([0.0, 0.0, 0.05, 0.001]), rng.random() < 0.5, rng.choice([0.1, 1.0, 3.0]))
    elif op == "norm":
        train = rng.random() < 0.7
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        c = groups * _log_int(rng, 1, max(1, 1024 // groups))
        h = _log_int(rng, 3, 160)  # from the 3x3 board on
        w = max(3, min(160, h + rng.choice([0, 0, 0, -1, 1, 5])))
        cap = (4 * 512 * 128 * 127 if train else 16384 * 64 * 225) // (c * h * w)
        n = _log_int(rng, 1, max(1, min(16384, cap)))
        case = _norm("", n, c, h, w, groups, rng.choice(list(DTYPES)), rng.choice(["none", "relu", "silu"]), rng.random() < 0.5, train)
    else:
        dtype = rng.choice(["f32", "bf16", "f16"])
        m = _log_int(rng, 1, 2048)
        k = _log_int(rng, 1, 4096)
        many = _log_int(rng, 1, max(1, min(24, 30_000_000_000 // (min(m, k) * min(m, k) * max(m, k) * 15))))
        terms = [f"{m}x{k}x{many}"]
        if rng.random() < 0.4:
            terms.append(f"{_log_int(rng, 1, 256)}x{_log_int(rng, 1, 600)}x{rng.randint(1, 3)}")
        case = _ortho("", " ".join(terms), dtype)
    del case["name"]
    return case


def _shapes(case):
    out = []
    for term in case["shapes"].split():
        m, k, many = (int(v) for v in term.split("x"))
        out += [(m, k)] * many
    return out


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "sample":
        rows, n = case["rows"], case["n"]
        st["scores"] = (randn(rows, n) * case["spread"]).to(dt)
        st["uniforms"] = torch.rand(rows, device="cuda", generator=g)
        st["temperature"] = case["temperature"]
        if case["temperature"] == "rows":  # the annealed temperatures of games of different age
            st["temperature"] = 0.1 + 0.9 * torch.rand(rows, device="cuda", generator=g)
        st["legal"] = (torch.rand(rows, n, device="cuda", generator=g) < 0.7) if case["legal"] else None
    elif case["op"] == "norm":
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]
        # channels last: what a convolution leaves, every channel with an offset and a scale of its own
        x = torch.empty(n, h, w, c, device="cuda", dtype=dt)
        off, sc = randn(c) * 0.5, 0.5 + torch.rand(c, device="cuda", generator=g)
        x.copy_(randn(n, h, w, c) * sc + off)
        st["x"] = x.permute(0, 3, 1, 2)
        st["weight"], st["bias"] = 1.0 + 0.2 * randn(c), 0.2 * randn(c)
        st["residual"] = randn(n, h, w, c).to(dt).permute(0, 3, 1, 2) if case["residual"] else None
        if case["train"]:
            st["dy"] = randn(n, h, w, c).to(dt).permute(0, 3, 1, 2)
            for k in ("x", "weight", "bias", "residual"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
    else:
        # gradients: a few strong directions over noise
        st["matrices"] = []
        for m, k in _shapes(case):
            r = min(m, k, 4)
            st["matrices"].append((randn(m, k) * 1e-3 + (randn(m, r) @ randn(r, k)) * (3e-3 / r)).to(dt))
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_sample(st):
    """in 64 bits: the drawn index depends on sums of many small weights and on values next to a border"""
    case = st["case"]
    s = st["scores"].double()
    rows, n = s.shape
    if st["legal"] is not None:
        s = torch.where(st["legal"], s, -math.inf)
    top = s.max(1, keepdim=True).values
    t = st["temperature"]
    t = t.double().view(-1, 1) if torch.is_tensor(t) else torch.full((rows, 1), t, dtype=torch.float64, device=s.device)
    w = torch.exp((s - top) / t.clamp(min=1e-300))
    w = torch.where(t > 0, w, (s == top).double())
    w = torch.where(top > -math.inf, w, torch.zeros_like(w))
    order = torch.sort(s, dim=1, descending=True, stable=True).indices
    ws = torch.gather(w, 1, order)
    rank = torch.arange(n, device=s.device).view(1, -1)
    k = case["top_k"] if 0 < case["top_k"] < n else n
    keep = (rank < k) & ((t > 0) | (rank == 0))
    ws = torch.where(keep, ws, 0.0)
    upto = torch.cumsum(ws, 1)
    if case["top_p"] < 1.0:
        keep = keep & ((upto - ws < case["top_p"] * upto[:, -1:]) | (rank == 0))
    keep = keep & (ws > 0) & (ws >= case["min_p"])
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    upto = torch.cumsum(kept, 1)
    target = st["uniforms"].double().view(-1, 1) * upto[:, -1:]
    hit = (upto > target) & (kept > 0)
    last = torch.where(kept > 0, rank, -1).max(1).values
    first = torch.where(hit, rank, n).min(1).values
    action = torch.where(first < n, first, last)
    at = action.clamp(min=0).view(-1, 1)
    some = (action >= 0).view(-1, 1)
    drop = torch.where(t > 0, (torch.gather(s, 1, at) - top) / t.clamp(min=1e-300), 0.0)
    logp = torch.where(some, drop - torch.log(upto[:, -1:]), -math.inf)
    return [action.to(torch.int32), logp.view(-1).float()]


def _plain_norm(st):
    case = st["case"]
    x, dt = st["x"].detach(), DTYPES[case["dtype"]]
    n, c, h, w = x.shape
    g, relu = case["groups"], case["act"] == "relu"
    # a gradient through relu hangs on the sign of values next to zero: those are decided in 64 bits
    acc = torch.float64 if case["train"] and relu else torch.float32

    def rows(t):
        return t.detach().permute(0, 2, 3, 1).reshape(n, h * w, g, c // g).to(acc)

    def planes(t):
        return t.reshape(n, h, w, c).to(dt).permute(0, 3, 1, 2)

    xs = rows(x)
    weight, bias = (st[k].detach().to(acc).view(1, 1, g, c // g) for k in ("weight", "bias"))
    mean = xs.mean((1, 3), keepdim=True)
    xc = xs - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean((1, 3), keepdim=True) + GN_EPS)
    xhat = xc * rstd
    z = xhat * weight + bias
    if st["residual"] is not None:
        z = z + rows(st["residual"])
    sig = torch.sigmoid(z) if case["act"] == "silu" else None
    y = z.clamp(min=0) if relu else z * sig if sig is not None else z
    if not case["train"]:
        return planes(y)
    dz = rows(st["dy"])
    if relu:
        dz = torch.where(z > 0, dz, 0.0)
    elif sig is not None:
        dz = dz * (sig * (1 + z * (1 - sig)))
    gx = dz * weight
    dx = rstd * (gx - gx.mean((1, 3), keepdim=True) - xhat * (gx * xhat).mean((1, 3), keepdim=True))
    out = [planes(y), planes(dx), (dz * xhat).sum((0, 1)).reshape(c).float(), dz.sum((0, 1)).reshape(c).float()]
    if st["residual"] is not None:
        out.append(planes(dz))
    return out


def _plain_ortho(st):
    a, b, c = NS_COEFFICIENTS
    out = []
    for m in st["matrices"]:
        x = m.float()
        tall = x.shape[0] > x.shape[1]
        x = x.t() if tall else x
        x = x / (torch.sqrt((x * x).sum()) + NS_EPS)
        for _ in range(5):
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
        out.append((x.t() if tall else x).to(m.dtype).contiguous())
    return out


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        return {"sample": _plain_sample, "norm": _plain_norm, "ortho": _plain_ortho}[case["op"]](state)
    from alphazero_amd import ops

    if case["op"] == "sample":
        return ops.sample_actions(state["scores"], state["uniforms"], temperature=state["temperature"], top_k=case["top_k"],
                                  top_p=case["top_p"], min_p=case["min_p"], legal=state["legal"], return_logprobs=True)
    if case["op"] == "norm":
        y = ops.group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], eps=GN_EPS, activation=case["act"],
                               residual=state["residual"])
        if not case["train"]:
            return y
        leaves = [state[k] for k in ("x", "weight", "bias", "residual") if state[k] is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
    return ops.orthogonalize(state["matrices"], steps=5, coefficients=NS_COEFFICIENTS, eps=NS_EPS)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "sample":
        e = case["rows"] * case["n"]
        per_row = 12 + (4 if case["temperature"] == "rows" else 0)
        return {"bytes": e * (b + (1 if case["legal"] else 0)) + case["rows"] * per_row, "flops": 4 * e}
    if case["op"] == "norm":
        e = case["n"] * case["c"] * case["h"] * case["w"]
        tensors = (2 + (1 if case["residual"] else 0)) if not case["train"] else (4 + (2 if case["residual"] else 0))
        return {"bytes": tensors * e * b + 4 * case["c"] * (4 if case["train"] else 2), "flops": e * (24 if case["train"] else 8)}
    by = fl = 0
    for m, k in _shapes(case):
        s, l = min(m, k), max(m, k)
        by += 2 * m * k * b
        fl += 5 * (3 * s * s * l + s * s * s)  # the two symmetric products count half
    return {"bytes": by, "flops": fl}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_sample(st):
    """row by row: walk the scores in descending order, then the kept ones in ascending index order"""
    case = st["case"]
    scores = st["scores"].float().cpu().numpy().astype(np.float64)
    u = st["uniforms"].cpu().numpy().astype(np.float64)
    legal = st["legal"].cpu().numpy() if st["legal"] is not None else None
    temp = st["temperature"]
    temp = temp.cpu().numpy().astype(np.float64) if torch.is_tensor(temp) else np.full(scores.shape[0], temp)
    out = np.full(scores.shape[0], -1, np.int32)
    logp = np.full(scores.shape[0], -np.inf)
    for r in range(scores.shape[0]):
        ids = np.flatnonzero(legal[r]) if legal is not None else np.arange(scores.shape[1])
        if ids.size == 0:
            continue
        s = scores[r, ids]
        if temp[r] <= 0:
            out[r], logp[r] = ids[np.argmax(s)], 0.0
            continue
        p = np.exp((s - s.max()) / temp[r])
        order = np.argsort(-s, kind="stable")
        if 0 < case["top_k"] < order.size:
            order = order[:case["top_k"]]
        sums = np.cumsum(p[order])
        if case["top_p"] < 1.0:  # the shortest run whose mass reaches top_p
            order = order[:1 + int(np.searchsorted(sums[:-1], case["top_p"] * sums[-1], side="left"))]
        order = order[p[order] >= case["min_p"]]
        kept = np.sort(order)
        sums = np.cumsum(p[kept])
        at = kept[min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), kept.size - 1)]
        out[r], logp[r] = ids[at], (s[at] - s.max()) / temp[r] - math.log(sums[-1])
    return [torch.from_numpy(out), torch.from_numpy(logp)]


def _exact_norm(st):
    """planes first, the gradients by differentiating the forward formula"""
    case = st["case"]
    leaves = {k: st[k].detach().double().contiguous() for k in ("x", "weight", "bias", "residual") if st[k] is not None}
    if case["train"]:
        for t in leaves.values():
            t.requires_grad_(True)
    x = leaves["x"]
    n, c, h, w = x.shape
    per = x.reshape(n, case["groups"], -1)
    mu = per.sum(2, keepdim=True) / per.shape[2]
    var = ((per - mu) ** 2).sum(2, keepdim=True) / per.shape[2]
    z = ((per - mu) / (var + GN_EPS).sqrt()).reshape(n, c, h * w) * leaves["weight"].view(1, c, 1) + leaves["bias"].view(1, c, 1)
    z = z.reshape(n, c, h, w)
    if "residual" in leaves:
        z = z + leaves["residual"]
    y = torch.relu(z) if case["act"] == "relu" else z / (1 + torch.exp(-z)) if case["act"] == "silu" else z
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), st["dy"].double())]


def _exact_ortho(st):
    """the polynomial applied to the Gram matrix of the other orientation: X <- X (aI + bS + cS^2), S = X^T X"""
    a, b, c = NS_COEFFICIENTS
    out = []
    for m in st["matrices"]:
        x = m.double()
        wide = x.shape[0] < x.shape[1]
        x = (x.t() if wide else x).contiguous()
        x = x / (x.pow(2).sum().sqrt() + NS_EPS)
        eye = torch.eye(x.shape[1], dtype=torch.float64, device=x.device)
        for _ in range(5):
            s = x.t() @ x
            x = x @ (a * eye + s @ (b * eye + c * s))
        out.append(x.t() if wide else x)
    return out


def exact(case, seed):
    if case["op"] == "sample" and case["rows"] * case["n"] > 48_000_000:
        return None
    st = prepare(case, seed)
    return {"sample": _exact_sample, "norm": _exact_norm, "ortho": _exact_ortho}[case["op"]](st)
