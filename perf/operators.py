"""W8A8 products and the router's balance loss, as cases that can be timed and compared.

  linear    linear_w8a8: rows of activations quantised to int8 with a scale per row, times an int8 matrix with a scale per channel -- the
            projections around the MoE layer in a W8A8 checkpoint
  experts   experts_w8a8: the routed experts of such a checkpoint behind the package's router: pairs sorted by expert (perm, offsets), rows
            gathered and quantised, gate / up product with the activation, quantised again, down product, rows back in pair order
  balance   balance_loss (evaluation) and balance_loss_grad (training): counts per expert, balance loss of each sequence, gradient of the logits

With own = False everything is computed from its formula with elementary torch operations; integer sums in 64 bits, so that they are exact.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_MOST_PRODUCT = 8192 * 4096 * 8192            # the largest listed linear case
_MOST_EXPERTS = 4096 * 8 * 512 * 2048 * 3     # ... and experts case, in multiplications
_MOST_WEIGHTS = 128 * 1856 * 2688 * 2         # ... and weights of one


def _linear(M, K, N, x, y, bias=False):
    return {"kind": "linear", "M": M, "K": K, "N": N, "x": x, "y": y, "bias": bias}


def _experts(T, H, F, E, k, act, x, zipf):
    return {"kind": "experts", "T": T, "H": H, "F": F, "E": E, "k": k, "act": act, "x": x, "y": "bf16", "zipf": zipf}


def _balance(S, L, E, k, x, mode, train, padded):
    return {"kind": "balance", "S": S, "L": L, "E": E, "k": k, "x": x, "mode": mode, "train": train, "padded": padded}


def listed():
    return [
        # one user's token through a projection of a 2048-wide model: latency
        {"name": "linear-1"} | _linear(1, 2048, 4096, "bf16", "bf16"),
        # seven slots through the up matrix of the Nemotron-H-style shared expert, f32 rows as the layer entries have them
        {"name": "linear-7"} | _linear(7, 2688, 3712, "f32", "f32", bias=True),
        # an almost full set of slots through an output projection
        {"name": "linear-61"} | _linear(61, 4096, 2048, "bf16", "bf16"),
        # a ragged prompt; sizes that are no multiple of anything
        {"name": "linear-777"} | _linear(777, 2005, 4099, "f16", "f16", bias=True),
        # the largest prompt chunk through a wide projection: the tensor pipe
        {"name": "linear-8192"} | _linear(8192, 4096, 8192, "bf16", "bf16"),
        # one token through eight of 256 experts
        {"name": "experts-1"} | _experts(1, 2048, 512, 256, 8, "swiglu", "bf16", False),
        # sixteen slots, most pairs on an expert of their own
        {"name": "experts-16"} | _experts(16, 2048, 512, 256, 8, "swiglu", "f32", False),
        # the Nemotron-H-style layer, a ragged prompt chunk: all experts touched, sixteen pairs each
        {"name": "experts-333-relu2"} | _experts(333, 2688, 1856, 128, 6, "relu2", "bf16", False),
        # a long prompt chunk with skewed routing: experts with thousands of pairs beside experts with none
        {"name": "experts-4096-zipf"} | _experts(4096, 2048, 512, 256, 8, "swiglu", "bf16", True),
        # counts and loss of a decode batch, as a monitor takes them
        {"name": "balance-24"} | _balance(1, 24, 256, 8, "f32", "softmax", False, False),
        # a padded training batch of four ragged sequences, sigmoid router
        {"name": "balance-4x1000"} | _balance(4, 1000, 128, 6, "bf16", "sigmoid", True, True),
        # a full training batch of long sequences
        {"name": "balance-16x8192"} | _balance(16, 8192, 256, 8, "f32", "softmax", True, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "experts", "balance"])
    if kind == "linear":
        while True:
            M, K, N = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
            if M * K * N <= _MOST_PRODUCT:
                return _linear(M, K, N, rng.choice(sorted(_TYPES)), rng.choice(sorted(_TYPES)), rng.random() < 0.5)
    if kind == "experts":
        while True:
            E, act = _log_int(rng, 4, 256), rng.choice(["swiglu", "relu2"])
            T, H, F = _log_int(rng, 1, 4096), _log_int(rng, 256, 2688), _log_int(rng, 64, 1856)
            k, m = rng.randint(1, min(8, E)), 3 if act == "swiglu" else 2
            if E * H * F * m <= _MOST_WEIGHTS and T * k * H * F * m <= _MOST_EXPERTS:
                return _experts(T, H, F, E, k, act, rng.choice(sorted(_TYPES)), rng.random() < 0.5)
    E = _log_int(rng, 4, 256)
    T = _log_int(rng, 1, 16 * 8192)
    S = _log_int(rng, 1, min(T, 64))
    return _balance(S, T // S, E, rng.randint(1, min(8, E)), rng.choice(sorted(_TYPES)), rng.choice(["softmax", "sigmoid"]), rng.random() < 0.7, rng.random() < 0.5)


# ---- inputs ----
def _int8(gen, *shape):
    """Weights ~N(0, 1) quantised by channel: the largest of some thousand values lies near four deviations.  Rows start on 16-byte boundaries."""
    K = shape[-1]
    q = torch.zeros(*shape[:-1], (K + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    if len(shape) == 2:
        q[:, :K] = torch.randn(shape, generator=gen, device="cuda").mul_(31).round_().clamp_(-127, 127)
    else:
        step = max(1, (1 << 26) // (shape[1] * K))
        for e in range(0, shape[0], step):
            part = q[e:e + step, :, :K]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda").mul_(31).round_().clamp_(-127, 127))
    return q[..., :K]


def _scales(gen, *shape):
    """Of weights ~N(0, 0.02): a channel's largest value over 127."""
    return 0.02 / 31 * (1 + 0.1 * torch.rand(shape, generator=gen, device="cuda"))


def _logits(gen, T, E, zipf):
    l = torch.randn(T, E, generator=gen, device="cuda") * 0.9
    if zipf:
        rank = torch.randperm(E, generator=gen, device="cuda") + 1
        l -= 2.2 * rank.float().log()
    return l


def prepare(case, seed):
    kind = case["kind"]
    size = case["M"] * 31 + case["K"] if kind == "linear" else case["T"] if kind == "experts" else case["S"] * 37 + case["L"]
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + size)
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"kind": kind, "x": torch.randn(M, K, generator=gen, device="cuda").to(_TYPES[case["x"]]), "w": _int8(gen, N, K), "sw": _scales(gen, N),
                "bias": torch.randn(N, generator=gen, device="cuda") * 0.1 if case["bias"] else None, "y": _TYPES[case["y"]]}
    if kind == "experts":
        T, H, F, E, k = case["T"], case["H"], case["F"], case["E"], case["k"]
        ids = _logits(gen, T, E, case["zipf"]).topk(k, dim=1).indices.reshape(-1)
        perm = torch.sort(ids, stable=True).indices.to(torch.int32)
        counts = torch.bincount(ids, minlength=E)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = counts.cumsum(0)
        rows = 2 * F if case["act"] == "swiglu" else F
        return {"kind": kind, "x": torch.randn(T, H, generator=gen, device="cuda").to(_TYPES[case["x"]]), "k": k, "act": case["act"], "y": _TYPES[case["y"]],
                "perm": perm, "offsets": offsets, "ends": offsets.tolist(),
                "w_up": _int8(gen, E, rows, H), "s_up": _scales(gen, E, rows), "w_down": _int8(gen, E, H, F), "s_down": _scales(gen, E, H)}
    S, L, E, k = case["S"], case["L"], case["E"], case["k"]
    logits = _logits(gen, S * L, E, True).to(_TYPES[case["x"]])
    ids = logits.float().topk(k, dim=1).indices.to(torch.int32)
    lengths = torch.randint(1, L + 1, (S,), generator=gen, device="cuda")
    mask = torch.arange(L, device="cuda") < lengths[:, None] if case["padded"] else None
    return {"kind": kind, "logits": logits.reshape(S, L, E), "ids": ids.reshape(S, L, k), "mask": mask, "mode": case["mode"], "train": case["train"]}


# ---- the plain forms ----
def _quantised(x):
    """Rows to whole numbers in [-127, 127] and a scale per row (a division by a number on the host would be a product with its reciprocal)."""
    x = x.float()
    a = x.abs().amax(dim=1)
    scale = torch.where(a > 0, (a / torch.full_like(a, 127.0)).clamp_min(2.0 ** -126), 0.0)
    q = torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]), 0.0)
    return q, scale


def _product(q, scale, w, sw):
    """Whole-number sums in 64 bits, scales in 32."""
    return (q.double() @ w.double().T).float() * scale[:, None] * sw


def _expert(q, scale, s, e):
    g = _product(q, scale, s["w_up"][e], s["s_up"][e])
    F = s["w_down"].shape[2]
    h = g[:, :F] / (1 + torch.exp(-g[:, :F])) * g[:, F:] if s["act"] == "swiglu" else g.clamp_min(0).square()
    return _product(*_quantised(h), s["w_down"][e], s["s_down"][e])


def _probabilities(l, mode):
    if mode == "sigmoid":
        l = l.clamp_max(0) - torch.log1p(torch.exp(-l.abs()))     # log of the sigmoid: its normalised values are a softmax of these
    e = torch.exp(l - l.amax(dim=-1, keepdim=True))
    return e / e.sum(dim=-1, keepdim=True)


def _balance_plain(s):
    l, ids = s["logits"].float(), s["ids"].long()
    S, L, E = l.shape
    k = ids.shape[2]
    there = torch.ones(S, L, dtype=torch.bool, device=l.device) if s["mask"] is None else s["mask"]
    p = torch.where(there[:, :, None], _probabilities(l, s["mode"]), 0.0)
    n = there.sum(dim=1)
    counts = torch.zeros(S, E, dtype=torch.int64, device=l.device).scatter_add_(1, ids.reshape(S, L * k), there[:, :, None].expand(S, L, k).reshape(S, L * k).long())
    prob = p.double().sum(dim=1) / n[:, None].clamp_min(1)
    c = E / (k * n.clamp_min(1).double())
    out = {"loss": (c * (counts * prob).sum(dim=1)).float(), "counts": counts.int(), "prob": prob.float(), "tokens": n.int()}
    if s["train"]:
        g = (c / n.clamp_min(1))[:, None] * (counts - counts.sum(dim=1, keepdim=True) / E)      # (the constant drops out below)
        g = g.float()[:, None, :]
        d = p * (g - (g * p).sum(dim=2, keepdim=True))
        if s["mode"] == "sigmoid":
            d = d / (1 + torch.exp(l))
        out["d_logits"] = torch.where(there[:, :, None], d, 0.0).to(s["logits"].dtype)
    return out


def _plain(s):
    if s["kind"] == "linear":
        y = _product(*_quantised(s["x"]), s["w"], s["sw"])
        return (y if s["bias"] is None else y + s["bias"]).to(s["y"])
    if s["kind"] == "experts":
        perm, ends = s["perm"].long(), s["ends"]
        q, scale = _quantised(s["x"])
        q, scale = q[perm // s["k"]], scale[perm // s["k"]]
        rows = torch.cat([_expert(q[a:b], scale[a:b], s, e) for e, (a, b) in enumerate(zip(ends, ends[1:])) if b > a]).to(s["y"])
        return torch.empty_like(rows).index_copy_(0, perm, rows)
    return _balance_plain(s)


# ---- the framework's operators ----
def _own(s):
    from chimere_b200 import abi, balance, w8a8
    if s["kind"] == "linear":
        return w8a8.linear_w8a8(s["x"], s["w"], s["sw"], bias=s["bias"], out_dtype=s["y"])
    if s["kind"] == "experts":
        act = abi.ACT_SWIGLU if s["act"] == "swiglu" else abi.ACT_RELU2
        return w8a8.experts_w8a8(s["x"], s["perm"], s["offsets"], s["k"], s["w_up"], s["s_up"], s["w_down"], s["s_down"], act=act, out_dtype=s["y"])
    mode = abi.ROUTE_SOFTMAX_RENORM if s["mode"] == "softmax" else abi.ROUTE_SIGMOID_NORM_SCALE
    if s["train"]:
        r, d = balance.balance_loss_grad(s["logits"], s["ids"], mask=s["mask"], route_mode=mode)
        return {"loss": r.loss, "counts": r.counts, "prob": r.prob, "tokens": r.tokens, "d_logits": d}
    r = balance.balance_loss(s["logits"], s["ids"], mask=s["mask"], route_mode=mode)
    return {"loss": r.loss, "counts": r.counts, "prob": r.prob, "tokens": r.tokens}


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ----
def work(case):
    kind = case["kind"]
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K * _SIZE[case["x"]] + N * K + (8 if case["bias"] else 4) * N + M * N * _SIZE[case["y"]], "flops": 2 * M * N * K}
    if kind == "experts":
        T, H, F, E, k = case["T"], case["H"], case["F"], case["E"], case["k"]
        m = 3 if case["act"] == "swiglu" else 2
        touched = E * (1 - (1 - k / E) ** T)      # experts with pairs, were the routing even
        if case["zipf"]:
            weight = [r ** -2.2 for r in range(1, E + 1)]
            total = sum(weight)
            touched = sum(1 - (1 - min(1.0, k * w / total)) ** T for w in weight)
        return {"bytes": int(T * H * _SIZE[case["x"]] + touched * (m * H * F + 4 * ((m - 1) * F + H)) + T * k * (H * _SIZE[case["y"]] + 4)), "flops": 2 * T * k * m * H * F}
    T, E, k = case["S"] * case["L"], case["E"], case["k"]
    return {"bytes": T * E * _SIZE[case["x"]] * (2 if case["train"] else 1) + T * (4 * k + (1 if case["padded"] else 0)) + case["S"] * (8 * E + 8), "flops": T * E * (12 if case["train"] else 6)}


# ---- the definition in 64 bits ----
def _exact_rows(x):
    """Scale and quotient are defined with one rounding to 32 bits each; from 64 bits that rounding is the same."""
    x = x.double()
    top = x.abs().max(dim=1, keepdim=True).values
    scale = (top / 127.0).float().double().clamp(min=2.0 ** -126)
    return torch.where(top > 0, (x / scale).float().double().round(), 0.0), torch.where(top > 0, scale, 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        q, scale = _exact_rows(s["x"])
        y = torch.matmul(q, s["w"].double().t()) * scale * s["sw"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["kind"] == "experts":
        token = torch.div(s["perm"].long(), case["k"], rounding_mode="floor")
        y = torch.zeros(case["T"] * case["k"], case["H"], dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            pairs = slice(s["ends"][e], s["ends"][e + 1])
            if pairs.start == pairs.stop:
                continue
            q, scale = _exact_rows(s["x"][token[pairs]])
            u = torch.matmul(q, s["w_up"][e].double().t()) * scale * s["s_up"][e].double()
            if case["act"] == "swiglu":
                gate, up = u.chunk(2, dim=1)
                h = gate * torch.sigmoid(gate) * up
            else:
                h = torch.relu(u) ** 2
            q, scale = _exact_rows(h.float())        # (the activations are held in 32 bits)
            y[s["perm"][pairs].long()] = torch.matmul(q, s["w_down"][e].double().t()) * scale * s["s_down"][e].double()
        return y
    l, E, k = s["logits"].double(), case["E"], case["k"]
    loss, counts, prob, tokens, grads = [], [], [], [], []
    for b in range(case["S"]):
        here = l[b] if s["mask"] is None else l[b][s["mask"][b]]
        ids = s["ids"][b] if s["mask"] is None else s["ids"][b][s["mask"][b]]
        n = here.shape[0]
        f = torch.bincount(ids.reshape(-1).long(), minlength=E)
        score = here if case["mode"] == "softmax" else torch.nn.functional.logsigmoid(here)
        p = torch.softmax(score, dim=1)
        mean = p.mean(dim=0)
        loss.append(E / (k * n) * (f.double() * mean).sum())
        counts.append(f)
        prob.append(mean)
        tokens.append(n)
        if case["train"]:
            f = f.double()
            d = E / (k * float(n) ** 2) * p * (f - (p @ f)[:, None])
            if case["mode"] == "sigmoid":
                d = d * torch.sigmoid(-here)
            full = torch.zeros_like(l[b])
            full[:n] = d
            grads.append(full)
    out = {"loss": torch.stack(loss), "counts": torch.stack(counts).int(), "prob": torch.stack(prob), "tokens": torch.tensor(tokens, dtype=torch.int32, device="cuda")}
    if case["train"]:
        out["d_logits"] = torch.stack(grads)
    return out
