"""The training operators around the logic layers, as measured cases: dropout from a counter-based generator, layer norm,
the log-probability of chosen actions, and the clipped policy loss with its KL term, forward and backward.

A case names the operator, the logical sizes (`n` rows: samples or tokens; `d` features, or `v` actions / classes / vocabulary
entries), the element type, the storage layout ("rows": a row's entries are contiguous; "features": the batch is contiguous,
the layout in which logic layers and the fused group sum hand over their outputs) and the direction ("forward", or "train":
the forward pass and its gradients).
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the output of a small hidden layer (96 neurons, batch 48): the call is all latency
        {"name": "dropout_small", "op": "dropout", "n": 48, "d": 96, "dtype": "float32", "layout": "features",
         "p": 0.1, "rescale": True, "way": "train"},
        # between two 64000-neuron layers at batch 1024, bf16 activations
        {"name": "dropout_wide", "op": "dropout", "n": 1024, "d": 64000, "dtype": "bfloat16", "layout": "features",
         "p": 0.1, "rescale": False, "way": "train"},
        # ragged sizes, rows that start on odd addresses, a high drop rate
        {"name": "dropout_odd", "op": "dropout", "n": 1001, "d": 16383, "dtype": "float16", "layout": "rows",
         "p": 0.5, "rescale": True, "way": "train"},
        # one observation of 784 features normalised for a decision
        {"name": "norm_single", "op": "norm", "n": 1, "d": 784, "dtype": "float32", "layout": "rows", "way": "forward"},
        # a batch of token features
        {"name": "norm_rows", "op": "norm", "n": 8192, "d": 4096, "dtype": "bfloat16", "layout": "rows", "way": "train"},
        # 16384 features of a convolutional stage at batch 512, in the layers' own layout
        {"name": "norm_features", "op": "norm", "n": 512, "d": 16384, "dtype": "float32", "layout": "features", "way": "train"},
        # ragged sizes, rows that start on odd addresses
        {"name": "norm_odd", "op": "norm", "n": 3001, "d": 5001, "dtype": "float16", "layout": "rows", "way": "train"},
        # what the behaviour policy thought of its actions: a batch of 10-class decisions out of the group sum
        {"name": "logp_actions", "op": "logp", "n": 1024, "v": 10, "dtype": "float32", "layout": "features", "way": "forward"},
        # log-probabilities of the tokens of a batch of sequences, with their gradient
        {"name": "logp_vocab", "op": "logp", "n": 4096, "v": 32768, "dtype": "bfloat16", "layout": "rows", "way": "train"},
        # a policy step on 10-class decisions out of the group sum, some actions forbidden
        {"name": "policy_actions", "op": "policy", "n": 1024, "v": 10, "dtype": "float32", "layout": "features",
         "masked": 0.1, "forbidden": True, "kl": True, "way": "train"},
        # a policy step on the tokens of a batch of sequences with a large vocabulary
        {"name": "policy_vocab", "op": "policy", "n": 2048, "v": 131072, "dtype": "bfloat16", "layout": "rows",
         "masked": 0.0, "forbidden": False, "kl": True, "way": "train"},
        # ragged sizes, rows that start on odd addresses, a third of the tokens padding
        {"name": "policy_odd", "op": "policy", "n": 1777, "v": 50001, "dtype": "float32", "layout": "rows",
         "masked": 0.33, "forbidden": False, "kl": True, "way": "train"},
    ]


def _log(rng, lo, hi):
    k = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return k + 1 if k == 3072 else k


def draw(rng):
    op = rng.choice(["dropout", "norm", "logp", "policy"])
    case = {"op": op, "dtype": rng.choice(sorted(DTYPES)), "layout": rng.choice(["rows", "features"])}
    case["way"] = "train" if op in ("dropout", "policy") else rng.choice(["forward", "train"])
    if op in ("dropout", "norm"):
        case["d"] = _log(rng, 96, 65536)
        case["n"] = _log(rng, 1, min(16384, (1 << 26) // case["d"]))
        if op == "dropout":
            case["p"] = rng.choice([0.05, 0.1, 0.25, 0.5])
            case["rescale"] = rng.choice([True, False])
    else:
        case["v"] = _log(rng, 2, 131072 if case["layout"] == "rows" else 1000)
        case["n"] = _log(rng, 64, min(65536, (1 << 26) // case["v"]))
        if op == "policy":
            case["masked"] = rng.choice([0.0, 0.1, 0.33])
            case["forbidden"] = rng.choice([True, False])
            case["kl"] = rng.choice([True, False])
    return case


# --------------------------------------------------------------------------------------------------------------- inputs
def _laid(n, d, layout, gen, make):
    """make(shape) in the case's layout, as a [n, d] tensor."""
    return make((n, d)) if layout == "rows" else make((d, n)).t()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    n, d, op = case["n"], case.get("d", case.get("v")), case["op"]

    def normal(shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    s = dict(case)
    if op == "dropout":
        s["x"] = _laid(n, d, case["layout"], g, lambda shape: torch.sigmoid(normal(shape)).to(dt))  # soft bits
        s["gy"] = _laid(n, d, case["layout"], g, lambda shape: normal(shape).to(dt))
        s["seed"], s["offset"] = 0x9E3779B97F4A + seed, 3 * seed + 1
    elif op == "norm":
        s["x"] = _laid(n, d, case["layout"], g, lambda shape: (normal(shape) * 1.5 + 0.5).to(dt))
        s["gy"] = _laid(n, d, case["layout"], g, lambda shape: normal(shape).to(dt))
        s["weight"] = 1 + 0.2 * normal((d,))
        s["bias"] = 0.2 * normal((d,))
        s["eps"] = 1e-5
    else:
        z = _laid(n, d, case["layout"], g, lambda shape: (2 * normal(shape)).to(dt))
        s["actions"] = torch.randint(0, d, (n,), generator=g, device="cuda")
        if case.get("forbidden"):
            shut = torch.rand(z.shape, generator=g, device="cuda") < 0.1
            shut.scatter_(1, s["actions"][:, None], False)
            z.masked_fill_(shut, float("-inf"))
            del shut
        s["x"] = z
        if op == "logp":
            s["gy"] = normal((n,)) / n
            s["temperature"] = 1.0
        else:
            rows = []
            for part, act in zip(z.split(256 if d > 4096 else 65536), s["actions"].split(256 if d > 4096 else 65536)):
                p = part.float()
                rows.append(p.gather(1, act[:, None])[:, 0] - torch.logsumexp(p, 1))
            logp = torch.cat(rows)
            # a policy some steps past the one that acted: ratios inside the clip range and beyond it, none on its edge
            step = torch.rand(n, generator=g, device="cuda") * 0.15
            step = torch.where(torch.rand(n, generator=g, device="cuda") < 0.3, step + 0.27, step)
            s["old_logp"] = logp + torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, -step, step)
            s["ref_logp"] = logp + 0.5 * normal((n,)) if case["kl"] else None
            s["advantages"] = normal((n,)) + 0.5
            s["mask"] = None
            if case["masked"]:
                s["mask"] = torch.rand(n, generator=g, device="cuda") >= case["masked"]
                s["actions"] = torch.where(s["mask"], s["actions"], -1)  # padding holds no action
            s["clip"], s["kl_coef"], s["temperature"] = 0.2, 0.05, 1.0
    if case["way"] == "train":
        s["x"] = s["x"].detach().requires_grad_()
        for k in ("weight", "bias"):
            if k in s:
                s[k] = s[k].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _philox_words(n, d, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): one counter for each 2 x 2 block of [n, d]; element (i, j) takes
    word 2 (i mod 2) + (j mod 2) of the block (i // 2, j // 2). int64 tensor [n, d] of 32-bit words."""
    low = 0xFFFFFFFF
    c0 = torch.arange((d + 1) // 2, device="cuda")[None, :].expand((n + 1) // 2, -1)
    c1 = torch.arange((n + 1) // 2, device="cuda")[:, None].expand(-1, (d + 1) // 2)
    c2, c3 = torch.full_like(c0, offset & low), torch.full_like(c0, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    w = torch.stack((torch.stack((c0, c1), -1), torch.stack((c2, c3), -1)), 1)  # [n/2, 2, d/2, 2]
    return w.reshape(w.shape[0] * 2, -1)[:n, :d]


def _plain_dropout(s):
    p = s["p"]
    keep = _philox_words(s["n"], s["d"], s["seed"], s["offset"]) >= int(round(p * 2 ** 32))
    scale = 1.0 / (1.0 - p) if s["rescale"] else 1.0

    def drop(t):
        return torch.where(keep, t.float() * scale, torch.zeros((), device=t.device)).to(t.dtype)

    return {"y": drop(s["x"]), "gx": drop(s["gy"])}


def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"], s["bias"]
    c = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + s["eps"])
    h = c * r
    out = {"y": (h * w + b).to(s["x"].dtype)}
    if s["way"] == "train":
        gy = s["gy"].float()
        t = gy * w
        out["gx"] = (r * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))).to(s["x"].dtype)
        out["gw"], out["gb"] = (gy * h).sum(0), gy.sum(0)
    return out


def _log_softmax(z, temperature):
    z = z.float() / temperature
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    return z, e / total, top + torch.log(total)


def _plain_logp(s):
    z, p, lse = _log_softmax(s["x"], s["temperature"])
    a = s["actions"][:, None]
    out = {"logp": (z.gather(1, a) - lse)[:, 0]}
    if s["way"] == "train":
        c = s["gy"][:, None] / s["temperature"]
        grad = -c * p
        out["gx"] = grad.scatter_add_(1, a, c).to(s["x"].dtype)
    return out


def _plain_policy(s):
    z, p, lse = _log_softmax(s["x"], s["temperature"])
    live = s["mask"] if s["mask"] is not None else torch.ones_like(s["actions"], dtype=torch.bool)
    zero = torch.zeros((), device=z.device)
    a = torch.where(live, s["actions"], 0)[:, None]
    logp = torch.where(live, (z.gather(1, a) - lse)[:, 0], zero)
    ratio = torch.where(live, torch.exp(logp - s["old_logp"]), zero)
    adv = s["advantages"]
    free, held = ratio * adv, ratio.clamp(1 - s["clip"], 1 + s["clip"]) * adv
    rows, slope = -torch.minimum(free, held), torch.where(free <= held, -adv * ratio, zero)
    kl = None
    if s["ref_logp"] is not None:
        gap = torch.where(live, s["ref_logp"] - logp, zero)
        kl = torch.exp(gap) - gap - 1
        rows, slope = rows + s["kl_coef"] * kl, slope + s["kl_coef"] * (1 - torch.exp(gap))
    count = live.sum().clamp(min=1)
    c = (torch.where(live, slope, zero) / count / s["temperature"])[:, None]
    grad = (-c * p).scatter_add_(1, a, c)
    grad = torch.where(live[:, None], grad, zero).to(s["x"].dtype)
    out = {"loss": torch.where(live, rows, zero).sum() / count, "logp": logp, "ratio": ratio, "gx": grad}
    if kl is not None:
        out["kl"] = kl
    return out


@torch.no_grad()
def _plain(s):
    return {"dropout": _plain_dropout, "norm": _plain_norm, "logp": _plain_logp, "policy": _plain_policy}[s["op"]](s)


# ----------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    import compactlogic_b200 as cl
    op, x, train = s["op"], s["x"], s["way"] == "train"
    if op == "dropout":
        y = cl.dropout(x, s["p"], seed=s["seed"], offset=s["offset"], rescale=s["rescale"])
        gx, = torch.autograd.grad(y, x, s["gy"])
        return {"y": y, "gx": gx}
    if op == "norm":
        y = cl.layer_norm(x, s["weight"], s["bias"], eps=s["eps"])
        if not train:
            return {"y": y}
        gx, gw, gb = torch.autograd.grad(y, (x, s["weight"], s["bias"]), s["gy"])
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    if op == "logp":
        logp = cl.action_log_probs(x, s["actions"], temperature=s["temperature"])
        if not train:
            return {"logp": logp}
        gx, = torch.autograd.grad(logp, x, s["gy"])
        return {"logp": logp, "gx": gx}
    r = cl.policy_loss(x, s["actions"], s["advantages"], s["old_logp"], ref_log_probs=s["ref_logp"], mask=s["mask"],
                       clip=s["clip"], kl_coef=s["kl_coef"], temperature=s["temperature"])
    gx, = torch.autograd.grad(r.loss, x)
    out = {"loss": r.loss, "logp": r.log_probs, "ratio": r.ratio, "gx": gx}
    if s["ref_logp"] is not None:
        out["kl"] = r.kl
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    n, e, train = case["n"], BYTES[case["dtype"]], case["way"] == "train"
    if case["op"] in ("dropout", "norm"):
        d = case["d"]
        nbytes = n * d * e * (4 if train else 2)
        if case["op"] == "norm":
            return {"bytes": nbytes + d * 4 * (4 if train else 2), "flops": n * d * (18 if train else 7)}
        return {"bytes": nbytes, "flops": 2 * n * d}
    v = case["v"]
    live = n * (1 - case.get("masked", 0.0))  # a padding row's logits need not be read
    nbytes = live * v * e + (n * v * e if train else 0) + n * 12
    if case["op"] == "policy":
        nbytes += n * (16 + (8 if case["kl"] else 0) + (1 if case["masked"] else 0))
    return {"bytes": int(nbytes), "flops": int(live * v * (8 if train else 4))}


# --------------------------------------------------------------------------------------------------- 64-bit definitions
def _exact_dropout(case, s):
    import numpy as np
    n, d, mask32 = case["n"], case["d"], np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    ctr = np.zeros(((n + 1) // 2, (d + 1) // 2, 4), np.uint64)
    ctr[..., 0] = np.arange((d + 1) // 2, dtype=np.uint64)[None, :]
    ctr[..., 1] = np.arange((n + 1) // 2, dtype=np.uint64)[:, None]
    ctr[..., 2], ctr[..., 3] = s["offset"] & 0xFFFFFFFF, s["offset"] >> 32
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    a, b, c, e = (np.ascontiguousarray(ctr[..., i]) for i in range(4))
    for r in range(10):
        ka = np.uint64((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF)
        kb = np.uint64((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF)
        lo, hi = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, e = (hi >> shift) ^ b ^ ka, hi & mask32, (lo >> shift) ^ e ^ kb, lo & mask32
    words = np.empty((2 * a.shape[0], 2 * a.shape[1]), np.uint64)
    words[0::2, 0::2], words[0::2, 1::2], words[1::2, 0::2], words[1::2, 1::2] = a, b, c, e
    kept = torch.from_numpy((words[:n, :d] / 2.0 ** 32 >= round(case["p"] * 2 ** 32) / 2.0 ** 32))
    factor = 1 / (1 - case["p"]) if case["rescale"] else 1.0
    kept = kept.to("cuda").double() * factor
    return {"y": s["x"].detach().double() * kept, "gx": s["gy"].double() * kept}


def _exact_norm(case, s):
    x = s["x"].detach().double()
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    std = torch.sqrt(var + s["eps"])
    out = {"y": (x - mean) / std * w + b}
    if case["way"] == "train":
        gy = s["gy"].double()
        hat = (x - mean) / std
        out["gw"], out["gb"] = torch.einsum("nd,nd->d", gy, hat), gy.sum(0)
        k = x.shape[1]
        back = gy * w
        out["gx"] = (k * back - back.sum(1, keepdim=True) - hat * (back * hat).sum(1, keepdim=True)) / (k * std)
    return out


def _exact_rows(case, s):
    """The losses by rows: the log-softmax of one block of rows at a time, and d loss / d logits = u (onehot - softmax)."""
    n, t = case["n"], s["temperature"]
    policy = case["op"] == "policy"
    live = torch.ones(n, dtype=torch.bool, device="cuda") if not policy or s["mask"] is None else s["mask"]
    count = max(1, int(live.sum()))
    got = {k: torch.zeros(n, dtype=torch.float64, device="cuda") for k in ("logp", "ratio", "kl", "loss")}
    grad = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda") if case["way"] == "train" else None
    block = max(1, (1 << 25) // case["v"])
    for i in range(0, n, block):
        at = torch.arange(i, min(n, i + block), device="cuda")[live[i:i + block]]
        if not at.numel():
            continue
        full = torch.log_softmax(s["x"].detach()[at].double() / t, dim=1)
        act = s["actions"][at]
        lp = full[torch.arange(at.numel(), device="cuda"), act]
        got["logp"][at] = lp
        if policy:
            adv, r = s["advantages"][at].double(), torch.exp(lp - s["old_logp"][at].double())
            lo, hi = 1 - s["clip"], 1 + s["clip"]
            open_ = torch.where(adv >= 0, r <= hi, r >= lo)
            loss, u = -adv * torch.where(open_, r, torch.where(adv >= 0, hi, lo).double()), torch.where(open_, -adv * r, 0.0)
            got["ratio"][at] = r
            if s["ref_logp"] is not None:
                q = s["ref_logp"][at].double() - lp
                kl = torch.expm1(q) - q
                got["kl"][at] = kl
                loss, u = loss + s["kl_coef"] * kl, u - s["kl_coef"] * torch.expm1(q)
            got["loss"][at] = loss / count
            u = u / count / t
        elif grad is not None:
            u = s["gy"][at].double() / t
        if grad is not None:
            g = -u[:, None] * torch.exp(full)
            g[torch.arange(at.numel(), device="cuda"), act] += u
            grad[at] = g
    out = {"logp": got["logp"]}
    if grad is not None:
        out["gx"] = grad
    if policy:
        out["loss"], out["ratio"] = got["loss"].sum(), got["ratio"]
        if s["ref_logp"] is not None:
            out["kl"] = got["kl"]
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"dropout": _exact_dropout, "norm": _exact_norm, "logp": _exact_rows, "policy": _exact_rows}[case["op"]](case, s)
