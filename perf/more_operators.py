"""Performance cases of the operators that serve many requests from one float model, and of its gated recurrence.

Three operators, each as a program calls it through ``mamba_int.ops``:

- ``sample_tokens``: the next token of every sequence from its logits, drawn with
  given random numbers after temperature, top-k, top-p and min-p;
- ``adapter_add``: low-rank adapters beside a shared projection, each sequence with
  its own adapter of a bank;
- ``gated_scan``: a gated linear recurrence over prompts and single tokens, with the
  gradients of its inputs, gates, decay and first state.

Sizes are those of ``bench.py``, ``perf/cases.py`` and the tests (d768 and d2048
models: d_inner 1536 and 4096, in_proj 2048 -> 8192, vocab 32000, prompts of
8 x 2048, decode batches of 8 and 64, the ragged BitLinear of 1000 -> 1108), a generic
vocabulary of 131072, and odd sizes between them.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "i8": torch.int8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i8": 1}
RATE = 8.0                      # the largest log decay of a gated step is RATE * softplus(decay)
LOGIT_SCALE = 1.0 / 4096.0      # what one unit of an integer logit stands for


def listed():
    return [
        # one sequence's next token with the usual filters: the smallest call
        {"name": "sample_one", "kind": "sample", "batch": 1, "vocab": 32000, "type": "f32", "temperature": 0.8,
         "top_k": 50, "top_p": 0.9, "min_p": 0.0, "rows": False},
        # a serving batch of the integer head's logits, every request with its own parameters
        {"name": "sample_requests", "kind": "sample", "batch": 64, "vocab": 32000, "type": "i32", "temperature": 1.0,
         "top_k": 40, "top_p": 0.95, "min_p": 0.05, "rows": True},
        # a serving batch over a large vocabulary in 16 bits (many equal logits), by mass alone
        {"name": "sample_wide", "kind": "sample", "batch": 64, "vocab": 131072, "type": "bf16", "temperature": 1.0,
         "top_k": 0, "top_p": 0.95, "min_p": 0.0, "rows": False},
        # out_proj of the d768 model for a decode step of eight requests
        {"name": "adapter_token", "kind": "adapter", "batch": 8, "len": 1, "k": 1536, "n": 768, "rank": 8, "bank": 16,
         "type": "f32", "weights": "bf16", "out": "f32", "lens": False, "none": 0.25},
        # in_proj of the d2048 model for a decode batch, nearly every request with another adapter
        {"name": "adapter_batch", "kind": "adapter", "batch": 64, "len": 1, "k": 2048, "n": 8192, "rank": 16, "bank": 128,
         "type": "bf16", "weights": "bf16", "out": "bf16", "lens": False, "none": 0.0},
        # out_proj of the d2048 model over a batch of prompts
        {"name": "adapter_prompt", "kind": "adapter", "batch": 8, "len": 2048, "k": 4096, "n": 2048, "rank": 32, "bank": 16,
         "type": "bf16", "weights": "bf16", "out": "bf16", "lens": False, "none": 0.0},
        # prompts of unequal lengths, 8-bit rows with their scales, an odd rank, requests without an adapter
        {"name": "adapter_ragged", "kind": "adapter", "batch": 5, "len": 333, "k": 1000, "n": 1108, "rank": 5, "bank": 7,
         "type": "i8", "weights": "f16", "out": "f32", "lens": True, "none": 0.4},
        # one decode step of the wide model's recurrence at a serving batch
        {"name": "gated_token", "kind": "gated", "batch": 64, "len": 1, "dim": 4096, "type": "bf16", "gate": True,
         "lens": False, "state": True, "train": False},
        # one layer over a batch of prompts
        {"name": "gated_prompt", "kind": "gated", "batch": 8, "len": 2048, "dim": 1536, "type": "bf16", "gate": True,
         "lens": False, "state": False, "train": False},
        # one long document: few channels, many steps
        {"name": "gated_long", "kind": "gated", "batch": 1, "len": 16384, "dim": 1536, "type": "f32", "gate": False,
         "lens": False, "state": True, "train": False},
        # a training step of one layer: the recurrence and its gradients
        {"name": "gated_train", "kind": "gated", "batch": 8, "len": 2048, "dim": 1536, "type": "bf16", "gate": True,
         "lens": False, "state": False, "train": True},
        # the same of sequences of unequal lengths (one empty) that continue from a state, odd sizes
        {"name": "gated_train_ragged", "kind": "gated", "batch": 3, "len": 701, "dim": 1003, "type": "f16", "gate": False,
         "lens": True, "state": True, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["sample", "sample", "adapter", "adapter", "gated", "gated", "gated"])
    if kind == "sample":
        vocab = rng.choice([32000, 131072, _log(rng, 500, 131072), _log(rng, 500, 131072)])
        return {"kind": kind, "batch": _log(rng, 1, min(256, 64 * 131072 // vocab)), "vocab": vocab,
                "type": rng.choice(["f32", "bf16", "f16", "i32"]), "temperature": rng.choice([1.0, round(rng.uniform(0.5, 1.5), 3)]),
                "top_k": rng.choice([0, 0, 1, _log(rng, 2, 1000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]), "rows": rng.random() < 0.5}
    if kind == "adapter":
        k = rng.choice([768, 1536, 2048, 4096, _log(rng, 200, 4096)])
        n = rng.choice([768, 2048, 8192, _log(rng, 200, 8192)])
        rank = rng.choice([4, 8, 16, 32, 64, _log(rng, 1, 64)])
        length = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
        typ = rng.choice(["f32", "bf16", "f16", "i8"])
        most = 8 * 2048 * 6144 * 32 // (length * (k + n) * max(rank, 32) * (1 if typ in ("bf16", "f16") else 2))
        batch = _log(rng, 1, max(1, min(64, most)))
        return {"kind": kind, "batch": batch, "len": length, "k": k, "n": n, "rank": rank, "bank": _log(rng, 1, 128),
                "type": typ, "weights": rng.choice(["f32", "bf16", "f16"]), "out": "f32" if typ == "i8" else typ,
                "lens": length > 1 and rng.random() < 0.3, "none": rng.choice([0.0, 0.3])}
    train = rng.random() < 0.5
    typ = rng.choice(["f32", "bf16", "f16"])
    dim = rng.choice([768, 1536, 2048, 4096, _log(rng, 100, 4096)])
    most = 8 * 2048 * 1536 * 2 // (5 if train and typ == "f32" else 2) // dim
    length = 1 if rng.random() < 0.2 else _log(rng, 2, min(16384, most))
    batch = _log(rng, 1, max(1, min(64, most // length)))
    return {"kind": kind, "batch": batch, "len": length, "dim": dim, "type": typ, "gate": rng.random() < 0.6,
            "lens": length > 1 and rng.random() < 0.25, "state": rng.random() < 0.5, "train": train}


# ------------------------------------------------------------------- inputs
def _lens(case, g):
    """Lengths of the sequences of a padded batch: one of them fills it, one is empty."""
    lens = torch.randint(0, case["len"] + 1, (case["batch"],), generator=g, device=DEV, dtype=torch.int32)
    lens[0] = case["len"]
    if case["batch"] > 2:
        lens[2] = 0
    return lens


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(shape, generator=g, device=DEV)

    s = {"case": case}
    kind, typ = case["kind"], TYPES[case["type"]]
    if kind == "sample":
        B, V = case["batch"], case["vocab"]
        # a language model's logits: falling with the token's rank, noise on top, in any order of tokens
        fall = torch.log(1.0 + torch.arange(V, device=DEV))[torch.randperm(V, generator=g, device=DEV)]
        logits = randn(B, V) - (0.6 + 0.8 * rand(B, 1)) * fall
        s["logits"] = torch.round(logits / LOGIT_SCALE).to(typ) if case["type"] == "i32" else logits.to(typ)
        s["scale"] = LOGIT_SCALE if case["type"] == "i32" else 1.0
        s["u"] = rand(B)
        for name in ("temperature", "top_k", "top_p", "min_p"):
            s[name] = case[name]
        if case["rows"]:       # requests with their own parameters: some greedy, some without a filter
            on = rand(4, B)
            s["temperature"] = torch.where(on[0] < 0.15, 0.0, case["temperature"] * (0.6 + 0.8 * rand(B)))
            s["top_k"] = torch.where(on[1] < 0.3, 0, torch.randint(1, 2 * case["top_k"] + 2, (B,), generator=g, device=DEV)).int()
            s["top_p"] = torch.where(on[2] < 0.3, 1.0, case["top_p"] * (0.6 + 0.4 * rand(B)))
            s["min_p"] = torch.where(on[3] < 0.5, 0.0, case["min_p"] * rand(B))
    elif kind == "adapter":
        B, L, K, N, r = (case[k] for k in ("batch", "len", "k", "n", "rank"))
        x = randn(B, L, K)
        if case["type"] == "i8":                              # the rows of an 8-bit norm, with their scales
            top = x.abs().amax(-1)
            s["x"] = torch.round(x * (127.0 / top).unsqueeze(-1)).to(torch.int8)
            s["x_scale"] = top / 127.0
        else:
            s["x"], s["x_scale"] = x.to(typ), None
        s["y"] = randn(B, L, N).to(TYPES[case["out"]])
        w = TYPES[case["weights"]]
        s["a"] = (randn(case["bank"], r, K) / math.sqrt(K)).to(w)
        s["b"] = (0.5 * randn(case["bank"], N, r) / math.sqrt(r)).to(w)
        s["scales"] = 0.5 + rand(case["bank"])
        ids = torch.randperm(max(case["bank"], B), generator=g, device=DEV)[:B] % case["bank"]
        s["ids"] = torch.where(rand(B) < case["none"], -1, ids).int()
        s["lens"] = _lens(case, g) if case["lens"] else None
        s["out"] = torch.empty_like(s["y"])
    else:
        B, L, D = case["batch"], case["len"], case["dim"]
        s["x"] = torch.nn.functional.silu(randn(B, L, D)).to(typ)
        ri = randn(B, L, 2 * D).to(typ)                       # both gates from one projection
        s["r"], s["i"] = ri[..., :D], ri[..., D:]
        s["z"] = randn(B, L, 2 * D).to(typ)[..., D:] if case["gate"] else None
        # a decay a = exp(-RATE * softplus(decay)) between 0.9 and 0.999 where the gate is open
        a = 0.9 + 0.099 * rand(D)
        s["decay"] = torch.log(torch.expm1(-torch.log(a) / RATE))
        s["lens"] = _lens(case, g) if case["lens"] else None
        s["h_in"] = randn(B, D) if case["state"] else None
        if case["train"]:
            s["dy"] = randn(B, L, D).to(typ)
        else:
            s["h_out"] = torch.empty((B, D), device=DEV)
    return s


# ------------------------------------------------- the framework's operators
def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba-integer_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mamba_int import ops
    return ops


def _run_own(s):
    ops, case = _ops(), s["case"]
    if case["kind"] == "sample":
        ids, logprob = ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                         min_p=s["min_p"], scale=s["scale"], logprob=True)
        return {"ids": ids, "logprob": logprob}
    if case["kind"] == "adapter":
        return ops.adapter_add(s["y"], s["x"], s["a"], s["b"], s["ids"], scales=s["scales"], x_scale=s["x_scale"],
                               lens=s["lens"], out=s["out"])
    if not case["train"]:
        y = ops.gated_scan(s["x"], s["r"], s["i"], s["decay"], z=s["z"], rate=RATE, h_in=s["h_in"], h_out=s["h_out"],
                           lens=s["lens"])
        return {"y": y, "h": s["h_out"]}
    names = [n for n in ("x", "r", "i", "decay", "z", "h_in") if s[n] is not None]
    leaf = {n: s[n].detach().requires_grad_() for n in names}
    y = ops.gated_scan(leaf["x"], leaf["r"], leaf["i"], leaf["decay"], z=leaf.get("z"), rate=RATE, h_in=leaf.get("h_in"),
                       lens=s["lens"])
    grads = torch.autograd.grad(y, [leaf[n] for n in names], s["dy"])
    return {"y": y.detach(), **{"d_" + n: d for n, d in zip(names, grads)}}


# --------------------------------------------------------------- plain forms
def _column(v, like):
    return (v if isinstance(v, torch.Tensor) else torch.tensor(v, device=DEV)).to(like.dtype).reshape(-1, 1)


def _plain_sample(s):
    """Filters by sorting, in 64 bits: every cut is a comparison of masses."""
    l = s["logits"].double() * s["scale"]
    V = l.shape[1]
    t, k = _column(s["temperature"], l), _column(s["top_k"], l)
    p, least = _column(s["top_p"], l), _column(s["min_p"], l)
    greedy = t <= 0
    top = l.amax(1, keepdim=True)
    e = (l - top) / torch.where(greedy, 1.0, t)
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    rank = torch.arange(V, device=DEV)
    w = torch.exp(e).gather(1, order)
    w = torch.where((k > 0) & (rank >= k), 0.0, w)
    mass = w.cumsum(1)
    total = mass[:, -1:]
    keep = (p >= 1) | (mass - w < p * total)              # what is before a token has not reached the mass
    keep = (keep & (w >= least) & (w > 0) & ~greedy) | (rank == 0)
    w = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))    # in the order of tokens
    mass = w.cumsum(1)
    total = mass[:, -1:]
    ids = (mass <= s["u"].double().unsqueeze(1) * total).sum(1, keepdim=True)
    ids = torch.minimum(ids, V - 1 - (w > 0).flip(1).int().argmax(1, keepdim=True))
    logprob = torch.log(w.gather(1, ids) / total)
    return {"ids": ids.squeeze(1), "logprob": logprob.squeeze(1).float()}


def _plain_adapter(s):
    B, L, _ = s["x"].shape
    ids = s["ids"].long()
    some = ids >= 0
    at = ids.clamp(min=0)
    x = s["x"].float()
    if s["x_scale"] is not None:
        x = x * s["x_scale"].unsqueeze(-1)
    t = torch.bmm(x, s["a"][at].float().transpose(1, 2).contiguous())
    t = t * torch.where(some, s["scales"][at], 0.0).view(B, 1, 1)
    if s["lens"] is not None:
        t = torch.where((torch.arange(L, device=DEV) < s["lens"].unsqueeze(1)).unsqueeze(-1), t, 0.0)
    d = torch.bmm(t, s["b"][at].float().transpose(1, 2).contiguous())
    return (s["y"].float() + d).to(s["y"].dtype)


def _scan(a, b):
    """h[t] = a[t] * h[t - 1] + b[t] along dimension 1 by doubling: after k rounds position t
    holds the decay and the input of the 2^k steps that end there."""
    L, k = a.shape[1], 1
    while k < L:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        if 2 * k < L:
            a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _plain_gated(s):
    case = s["case"]
    typ = s["x"].dtype
    x, sr, si = s["x"].float(), torch.sigmoid(s["r"].float()), torch.sigmoid(s["i"].float())
    B, L, D = x.shape
    soft = torch.clamp(s["decay"], min=0.0) + torch.log1p(torch.exp(-s["decay"].abs()))
    neg = RATE * soft * sr                                # minus the step's log decay
    a, m = torch.exp(-neg), torch.sqrt(-torch.expm1(-2.0 * neg))
    b = m * si * x
    keep = None
    if s["lens"] is not None:
        keep = (torch.arange(L, device=DEV) < s["lens"].unsqueeze(1)).unsqueeze(-1)
        a, b = torch.where(keep, a, 1.0), torch.where(keep, b, 0.0)
    first = s["h_in"] if s["h_in"] is not None else torch.zeros(B, D, device=DEV)
    h = _scan(a, torch.cat([b[:, :1] + a[:, :1] * first.unsqueeze(1), b[:, 1:]], 1))
    gate = torch.ones_like(h) if s["z"] is None else torch.sigmoid(s["z"].float())
    act = gate if s["z"] is None else gate * s["z"].float()
    y = h * act
    if keep is not None:
        y = torch.where(keep, y, 0.0)
    if not case["train"]:
        return {"y": y.to(typ), "h": h[:, -1].contiguous()}
    dy = s["dy"].float()
    if keep is not None:
        dy = torch.where(keep, dy, 0.0)
    # from the last step back: g[t] = act[t] dy[t] + a[t + 1] g[t + 1]
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _scan(after.flip(1), (act * dy).flip(1)).flip(1)
    before = torch.cat([first.unsqueeze(1), h[:, :-1]], 1)
    dneg = g * (si * x * a * a / m - a * before) * neg    # times neg: the gradient of log(neg)
    out = {"y": y.to(typ), "d_x": g * m * si, "d_r": dneg * (1.0 - sr), "d_i": g * b * (1.0 - si)}
    if keep is not None:
        dneg = torch.where(keep, dneg, 0.0)
        out = {n: torch.where(keep, v, 0.0) for n, v in out.items()}
    if s["z"] is not None:
        out["d_z"] = dy * h * (gate + act * (1.0 - gate))
        if keep is not None:
            out["d_z"] = torch.where(keep, out["d_z"], 0.0)
    out = {n: v.to(typ) for n, v in out.items()}
    out["d_decay"] = (dneg.double().sum((0, 1)) * torch.sigmoid(s["decay"].double()) / soft.double()).float()
    if s["h_in"] is not None:
        out["d_h_in"] = a[:, 0] * g[:, 0]
    return out


def run(s):
    if own:
        return _run_own(s)
    return {"sample": _plain_sample, "adapter": _plain_adapter, "gated": _plain_gated}[s["case"]["kind"]](s)


# ---------------------------------------------------------------- 64 bits
def _exact_sample(s):
    """Row by row: a kept token is one with few enough tokens, and little enough mass, in front of it."""
    import numpy as np
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    B, V = logits.shape
    par = {n: np.broadcast_to(v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.float64(np.float32(v)), (B,))
           for n, v in ((n, s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))}
    ids, logprob = np.zeros(B, np.int64), np.zeros(B)
    for b in range(B):
        l = logits[b] * s["scale"]
        if par["temperature"][b] <= 0:
            ids[b] = int(np.flatnonzero(l == l.max())[0])
            continue
        w = np.exp((l - l.max()) / par["temperature"][b])
        order = np.lexsort((np.arange(V), -l))            # by logit, then by token
        k = int(par["top_k"][b])
        if 0 < k < V:
            order = order[:k]
        total = math.fsum(w[order])
        n, mass = 0, 0.0
        for j in order.tolist():
            if n and ((par["top_p"][b] < 1 and mass >= par["top_p"][b] * total) or w[j] < par["min_p"][b]):
                break
            n, mass = n + 1, mass + w[j]
        kept = np.sort(order[:n])
        run = np.cumsum(w[kept].astype(np.longdouble))
        at = min(int(np.searchsorted(run, np.longdouble(u[b]) * run[-1], side="right")), n - 1)
        ids[b], logprob[b] = kept[at], float(np.log(w[kept[at]] / run[-1]))
    return {"ids": torch.from_numpy(ids), "logprob": torch.from_numpy(logprob)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "sample":
        return _exact_sample(s)
    if kind == "adapter":
        out = s["y"].double()
        for b in range(case["batch"]):
            j = int(s["ids"][b])
            n = int(s["lens"][b]) if s["lens"] is not None else case["len"]
            if j < 0 or n == 0:
                continue
            x = s["x"][b, :n].double()
            if s["x_scale"] is not None:
                x = x * s["x_scale"][b, :n, None].double()
            w = s["b"][j].double() @ s["a"][j].double()       # the adapter as one matrix
            out[b, :n] += s["scales"][j].double() * (x @ w.t())
        return out
    B, L, D = case["batch"], case["len"], case["dim"]
    if case["train"] and L * B * D > 30_000_000:
        return None
    names = [n for n in ("x", "r", "i", "decay", "z", "h_in") if s[n] is not None]
    v = {n: s[n].double().clone().requires_grad_(case["train"]) for n in names}
    zero = torch.zeros(B, D, dtype=torch.float64, device=DEV)
    h, ys = v.get("h_in", zero), []
    k = RATE * torch.logaddexp(v["decay"], torch.zeros_like(v["decay"]))
    rows = {n: v[n].unbind(1) for n in ("x", "r", "i", "z") if n in v}
    for t in range(L):
        log_a = -k / (1.0 + torch.exp(-rows["r"][t]))
        new = torch.exp(log_a) * h + torch.sqrt(-torch.expm1(2.0 * log_a)) * rows["x"][t] / (1.0 + torch.exp(-rows["i"][t]))
        out = new * rows["z"][t] / (1.0 + torch.exp(-rows["z"][t])) if "z" in rows else new
        if s["lens"] is not None:
            on = (s["lens"] > t).unsqueeze(1)
            new, out = torch.where(on, new, h), torch.where(on, out, 0.0)
        h = new
        ys.append(out)
    y = torch.stack(ys, 1)
    if not case["train"]:
        return {"y": y, "h": h}
    grads = torch.autograd.grad(y, [v[n] for n in names], s["dy"].double())
    return {"y": y.detach(), **{"d_" + n: d for n, d in zip(names, grads)}}


# ------------------------------------------------------------------- work
def work(case):
    kind, e = case["kind"], SIZE[case["type"]]
    if kind == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * e + case["batch"] * 32, "flops": 10 * n}
    if kind == "adapter":
        M, K, N, r = case["batch"] * case["len"], case["k"], case["n"], case["rank"]
        # each adapter that is used is read once
        used = min(case["batch"], case["bank"])
        weights = used * r * (K + N) * SIZE[case["weights"]]
        return {"bytes": M * (K * e + 2 * N * SIZE[case["out"]]) + weights, "flops": 2 * M * r * (K + N)}
    n = case["batch"] * case["len"] * case["dim"]
    gate = 1 if case["gate"] else 0
    states = 4 * case["batch"] * case["dim"] * (2 if case["state"] else 1)
    if case["train"]:
        # read: x, r, i, z, dy; written: y and the four gradients
        return {"bytes": n * e * (8 + 2 * gate) + states + 8 * case["dim"], "flops": n * (60 + 20 * gate)}
    return {"bytes": n * e * (4 + gate) + states + 4 * case["dim"], "flops": n * (25 + 6 * gate)}
