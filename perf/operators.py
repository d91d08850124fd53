"""What is measured of the sequence-training operators: the gated linear recurrence
(`gated_scan`, `scan_last`), the log-probabilities of chosen tokens (`token_logprob`), the
clipped policy loss with a KL term (`policy_loss`) and the preference loss of answer pairs
(`preference_loss`), each forward and, where a model trains through it, backward.

`run` computes a case in its plain form (elementary torch operations) or, with `own` set,
through the compiled programs of tinytensor_b200.  All data is float32, token ids int32.
"""

import math

import numpy as np
import torch

own = False

# Programs compiled so far, by the case's sizes and options: a training or serving program
# compiles once per shape and runs the result on every batch.
_PROGRAMS = {}


# ---- cases -----------------------------------------------------------------------------


def _scan(name, B, T, D, heads=0, axis=-2, init=False, train=True):
    c = {"op": "scan", "B": B, "T": T, "D": D, "heads": heads, "axis": axis, "init": init, "train": train}
    return {"name": name, **c} if name else c


def _logprob(name, B, T, V, train):
    c = {"op": "logprob", "B": B, "T": T, "V": V, "train": train}
    return {"name": name, **c} if name else c


def _policy(name, B, T, V, kl, lo=0.2, hi=0.2, per_token=True):
    c = {"op": "policy", "B": B, "T": T, "V": V, "kl": kl, "lo": lo, "hi": hi, "per_token": per_token}
    return {"name": name, **c} if name else c


def _preference(name, N, T, V, beta=0.1, smoothing=0.0):
    c = {"op": "preference", "B": N, "T": T, "V": V, "beta": beta, "smoothing": smoothing}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token for each of 64 running sequences, from their states: latency counts
        _scan("scan_step", 64, 1, 4096, init=True, train=False),
        # reading one long document: few channels for the card, many steps
        _scan("scan_prefill_long", 1, 65536, 1024, train=False),
        # a training step of a recurrent layer, states carried over from the last window
        _scan("scan_train", 8, 2048, 1024, init=True),
        # one gate for all channels of a head, broadcast, its gradient summed over the head
        _scan("scan_train_heads", 4, 2048, 1024, heads=16),
        # channels before time (the layout a convolution before the layer leaves), odd sizes
        _scan("scan_train_lines", 4, 8191, 500, axis=-1),
        # scoring the last token of a few requests over a large vocabulary
        _logprob("logprob_score", 8, 1, 131072, train=False),
        # cross-entropy training over an odd vocabulary (a size one past a multiple of 32)
        _logprob("logprob_train", 8, 512, 32001, train=True),
        # a policy step on 16 answers with prompts and padding masked, KL to a reference
        _policy("policy_train", 16, 512, 32768, kl=0.05),
        # a toy policy, one advantage for a whole answer: latency counts
        _policy("policy_small", 2, 64, 1000, kl=0.0, per_token=False),
        # odd sizes throughout, asymmetric clipping
        _policy("policy_ragged", 7, 311, 50001, kl=0.02, lo=0.2, hi=0.28, per_token=False),
        # eight pairs of answers
        _preference("preference_train", 8, 512, 16384),
        # a few short pairs over a small vocabulary, label smoothing
        _preference("preference_small", 3, 37, 257, smoothing=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "logprob", "policy", "preference"])
    if op == "scan":
        T = _log_int(rng, 1, 65536)
        heads = rng.choice([0, 0, 1, 3, 8])
        limit = (1 << 24) // T  # lanes, so that a drawn case stays below the largest listed one
        D = _log_int(rng, min(24, limit), min(4096, limit))
        if heads:
            D = heads * max(1, D // heads)
        B = _log_int(rng, 1, max(1, min(64, limit // D)))
        axis = -2 if heads else rng.choice([-2, -2, -1])
        return _scan(None, B, T, D, heads, axis, rng.random() < 0.5, rng.random() < 0.6)
    V = _log_int(rng, 200, 131072)
    rows = _log_int(rng, 8, min(8192, (1 << 27) // V))
    if op == "preference":
        rows = max(1, rows // 2)
    T = _log_int(rng, 1, rows)
    B = max(1, rows // T)
    if op == "logprob":
        return _logprob(None, B, T, V, rng.random() < 0.7)
    if op == "policy":
        return _policy(None, B, T, V, rng.choice([0.0, 0.01, 0.1]), rng.choice([0.1, 0.2]), rng.choice([0.2, 0.3]),
                       rng.random() < 0.5)
    return _preference(None, B, T, V, rng.choice([0.05, 0.1, 0.5]), rng.choice([0.0, 0.1]))


# ---- inputs ------------------------------------------------------------------------------


def _rows_shape(case):
    return (case["B"], 2, case["T"]) if case["op"] == "preference" else (case["B"], case["T"])


def _valid(case):
    """Which tokens count: prompts and the padding behind an answer do not, and with four or
    more sequences one of them is empty.  A function of the sizes alone, so that the work of
    a case does not depend on the seed."""
    shape = _rows_shape(case)
    n, T = int(np.prod(shape[:-1])), shape[-1]
    s = np.arange(n)[:, None]
    t = np.arange(T)[None, :]
    v = (t >= s * 37 % (T // 4 + 1)) & (t < T - s * 53 % (T // 8 + 1))
    if n >= 4 and T > 1:
        v[n // 2] = False
    return v.reshape(shape)


def _scan_inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    B, T, D, heads = case["B"], case["T"], case["D"], case["heads"]

    def normal(*s):
        return torch.randn(s, generator=g, device="cuda", dtype=torch.float32)

    if heads:
        full, gate_shape, lane = (B, T, heads, D // heads), (B, T, heads, 1), (B, heads, D // heads)
    elif case["axis"] == -1:
        full, gate_shape, lane = (B, D, T), (B, D, T), (B, D)
    else:
        full, gate_shape, lane = (B, T, D), (B, T, D), (B, D)
    # gates as a sigmoid leaves them, most near one; a few are zero, where a packed batch
    # starts its next document
    gate = torch.sigmoid(3.0 + 1.5 * normal(*gate_shape))
    gate = torch.where(torch.rand(gate_shape, generator=g, device="cuda") < 0.002, torch.zeros_like(gate), gate)
    d = {"gate": gate, "x": normal(*full)}
    if case["init"]:
        d["init"] = normal(*lane)
    if case["train"]:
        d["dh"] = normal(*full)
    return d


def _token_inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    shape, V = _rows_shape(case), case["V"]

    def normal(*s):
        return torch.randn(s, generator=g, device="cuda", dtype=torch.float32)

    logits = 2.5 * normal(*shape, V)
    tokens = torch.randint(0, V, shape, generator=g, device="cuda", dtype=torch.int32)
    valid = torch.from_numpy(_valid(case)).cuda()
    idx = tokens.long().unsqueeze(-1)
    lp = (logits.gather(-1, idx) - torch.logsumexp(logits, -1, keepdim=True)).squeeze(-1)
    tokens = torch.where(valid, tokens, torch.full_like(tokens, -1))
    d = {"logits": logits, "tokens": tokens}
    weight = valid.float() / max(1, int(_valid(case).sum()))
    if case["op"] == "logprob":
        if case["train"]:
            d["seed"] = -weight
        return d
    if case["op"] == "policy":
        # the sampling policy is a few updates old; ratios keep off the clip borders, where
        # the gradient jumps
        ratio = torch.exp(0.2 * normal(*shape))
        for border in (1.0 - case["lo"], 1.0 + case["hi"]):
            ratio = torch.where((ratio - border).abs() < 2e-3, ratio + 5e-3, ratio)
        d["old"] = lp - torch.log(ratio)
        d["advantage"] = normal(*shape) if case["per_token"] else normal(shape[0], 1)
        if case["kl"] > 0:
            d["ref"] = lp + 0.3 * normal(*shape)
        d["seed"] = weight
        return d
    d["ref"] = lp + 0.3 * normal(*shape)
    d["seed"] = torch.full((shape[0],), 1.0 / shape[0], device="cuda")
    return d


def _inputs(case, seed):
    return _scan_inputs(case, seed) if case["op"] == "scan" else _token_inputs(case, seed)


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"case": case, "in": d}
    if own:
        prog = _program(case, d)
        state["prog"] = prog
        state["args"] = list(d.values())
        state["outs"] = [torch.empty(s, device="cuda", dtype=torch.float32) for s in prog.output_shapes]
    return state


def _program(case, d):
    """The compiled program of a case: graph inputs in the order of `_inputs`."""
    import tinytensor_b200 as tt

    key = tuple(sorted((k, v) for k, v in case.items() if k != "name"))
    if key in _PROGRAMS:
        return _PROGRAMS[key]
    g = tt.Graph()
    n = {k: g.input(list(v.shape), dtype=tt.int32 if v.dtype == torch.int32 else tt.float32, name=k)
         for k, v in d.items()}
    if case["op"] == "scan":
        h = tt.gated_scan(n["gate"], n["x"], init=n.get("init"), axis=1 if case["axis"] == -2 else 2)
        if case["train"]:
            wrt = [n["gate"], n["x"]] + ([n["init"]] if case["init"] else [])
            prog = tt.compile_gradients(g, h, wrt, outputs=[h], seed=n["dh"])
        else:
            prog = tt.compile(g, [h, tt.scan_last(h)])
    else:
        if case["op"] == "logprob":
            y = tt.token_logprob(n["logits"], n["tokens"])
        elif case["op"] == "policy":
            y = tt.policy_loss(n["logits"], n["tokens"], n["old"], n["advantage"], ref_logp=n.get("ref"),
                               clip=(case["lo"], case["hi"]), kl=case["kl"])
        else:
            y = tt.preference_loss(n["logits"], n["tokens"], n["ref"], beta=case["beta"], smoothing=case["smoothing"])
        if "seed" in n:
            prog = tt.compile_gradients(g, y, [n["logits"]], outputs=[y], seed=n["seed"])
        else:
            prog = tt.compile(g, [y])
    _PROGRAMS[key] = prog
    return prog


# ---- one pass ------------------------------------------------------------------------------


def run(state):
    if own:
        state["prog"].run_device([t.data_ptr() for t in state["args"]], [t.data_ptr() for t in state["outs"]],
                                 stream=torch.cuda.current_stream().cuda_stream)
        return state["outs"]
    case, d = state["case"], state["in"]
    return _plain_scan(case, d) if case["op"] == "scan" else _plain_tokens(case, d)


def _doubling(a, x, dim):
    """h_t = a_t * h_{t-1} + x_t (h_{-1} = 0) in log2(T) steps: after the step of distance d,
    (a, h) of a position stand for the window of the 2d positions that end there."""
    T, d = x.shape[dim], 1
    while d < T:
        a0, a1 = a.narrow(dim, 0, T - d), a.narrow(dim, d, T - d)
        h1 = x.narrow(dim, d, T - d) + a1 * x.narrow(dim, 0, T - d)
        x = torch.cat([x.narrow(dim, 0, d), h1], dim)
        a = torch.cat([a.narrow(dim, 0, d), a0 * a1], dim)
        d *= 2
    return x


def _plain_scan(case, d):
    dim = 1 if case["axis"] == -2 else 2
    x, T = d["x"], case["T"]
    gate = d["gate"].expand_as(x)
    if case["init"]:
        first = x.narrow(dim, 0, 1) + gate.narrow(dim, 0, 1) * d["init"].unsqueeze(dim)
        x = torch.cat([first, x.narrow(dim, 1, T - 1)], dim)
    h = _doubling(gate, x, dim)
    if not case["train"]:
        return [h, h.select(dim, T - 1).clone()]
    # backward: u_t = dh_t + a_{t+1} * u_{t+1} is dx; da_t = u_t * h_{t-1}; dinit = a_0 * u_0
    zero = torch.zeros_like(x.narrow(dim, 0, 1))
    nxt = torch.cat([gate.narrow(dim, 1, T - 1), zero], dim)
    u = _doubling(nxt.flip(dim), d["dh"].flip(dim), dim).flip(dim)
    before = d["init"].unsqueeze(dim) if case["init"] else zero
    da = u * torch.cat([before, h.narrow(dim, 0, T - 1)], dim)
    if case["heads"]:
        da = da.sum(-1, keepdim=True)
    out = [h, da, u]
    if case["init"]:
        out.append((gate * u).select(dim, 0))
    return out


def _plain_tokens(case, d):
    logits, tokens = d["logits"], d["tokens"]
    valid = tokens >= 0
    idx = tokens.clamp(min=0).long().unsqueeze(-1)
    top = logits.max(-1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    # log-probabilities in 64 bits: their differences decide which side of a clip they are on
    lp = ((logits.gather(-1, idx) - top).double() - torch.log(total)).squeeze(-1)
    zero = torch.zeros_like(lp)
    lp = torch.where(valid, lp, zero)
    if case["op"] == "logprob":
        y, slope = lp, torch.where(valid, torch.ones_like(lp), zero)
    elif case["op"] == "policy":
        adv = d["advantage"].double()
        ratio = torch.exp(lp - d["old"].double())
        plain, held = ratio * adv, ratio.clamp(1.0 - case["lo"], 1.0 + case["hi"]) * adv
        y = -torch.minimum(plain, held)
        slope = torch.where(plain <= held, -plain, zero)
        if case["kl"] > 0:
            back = d["ref"].double() - lp
            y = y + case["kl"] * (torch.exp(back) - back - 1.0)
            slope = slope + case["kl"] * (1.0 - torch.exp(back))
        y, slope = torch.where(valid, y, zero), torch.where(valid, slope, zero)
    else:
        diff = torch.where(valid, lp - d["ref"].double(), zero).sum(-1)
        z = case["beta"] * (diff[:, 0] - diff[:, 1])
        eps = case["smoothing"]
        soft = torch.log1p(torch.exp(-z.abs()))
        y = (1.0 - eps) * (soft + (-z).clamp(min=0)) + eps * (soft + z.clamp(min=0))
        p = 1.0 / (1.0 + torch.exp(-z))
        dz = (eps * p - (1.0 - eps) * (1.0 - p)) * case["beta"]
        slope = torch.stack([dz, -dz], 1).unsqueeze(-1) * valid
    if "seed" not in d:
        return [y.float()]
    seed = d["seed"].double()
    if case["op"] == "preference":
        seed = seed[:, None, None]
    c = (seed * slope).float().unsqueeze(-1)
    dlogits = e * (-c / total.float())
    dlogits.scatter_add_(-1, idx, c)
    # what a padded position holds has no share in the gradient, whatever it is
    return [y.float(), torch.where(valid.unsqueeze(-1), dlogits, torch.zeros_like(dlogits))]


# ---- the definition in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    d = _inputs(case, seed)
    return _exact_scan(case, d) if case["op"] == "scan" else _exact_tokens(case, d)


def _exact_scan(case, d):
    dim = 1 if case["axis"] == -2 else 2
    x = d["x"].double().movedim(dim, 0).contiguous()
    a = d["gate"].double().expand(d["x"].shape).movedim(dim, 0).contiguous()
    h = torch.empty_like(x)
    s = d["init"].double() if case["init"] else torch.zeros_like(x[0])
    for t in range(case["T"]):
        s = torch.addcmul(x[t], a[t], s)
        h[t] = s
    hout = h.movedim(0, dim)
    if not case["train"]:
        return [hout, s]
    u = d["dh"].double().movedim(dim, 0).contiguous()
    for t in range(case["T"] - 2, -1, -1):
        u[t].addcmul_(a[t + 1], u[t + 1])
    da = torch.empty_like(h)
    da[1:] = u[1:] * h[:-1]
    da[0] = u[0] * d["init"].double() if case["init"] else 0.0
    da = da.movedim(0, dim)
    out = [hout, da.sum(-1, keepdim=True) if case["heads"] else da, u.movedim(0, dim)]
    if case["init"]:
        out.append(a[0] * u[0])
    return out


def _exact_tokens(case, d):
    shape, V = _rows_shape(case), case["V"]
    rows = int(np.prod(shape))
    logits = d["logits"].reshape(rows, V)
    tokens = d["tokens"].reshape(rows).long()
    live = torch.nonzero(tokens >= 0).squeeze(-1)
    lp = torch.zeros(rows, dtype=torch.float64, device="cuda")
    for part in live.split(512):
        full = torch.log_softmax(logits[part].double(), -1)
        lp[part] = full[torch.arange(len(part), device="cuda"), tokens[part]]
    dead = tokens < 0
    if case["op"] == "logprob":
        y, slope = lp, torch.ones_like(lp)
    elif case["op"] == "policy":
        adv = d["advantage"].double().expand(shape).reshape(rows)
        r = torch.exp(lp - d["old"].double().reshape(rows))
        high, low = r > 1.0 + case["hi"], r < 1.0 - case["lo"]
        held = torch.where(high, torch.full_like(r, 1.0 + case["hi"]), torch.where(low, torch.full_like(r, 1.0 - case["lo"]), r))
        y = torch.where(r * adv < held * adv, -r * adv, -held * adv)
        stopped = (high & (adv > 0)) | (low & (adv < 0))
        slope = torch.where(stopped, torch.zeros_like(r), -adv * r)
        if case["kl"] > 0:
            k = d["ref"].double().reshape(rows) - lp
            y = y + case["kl"] * (torch.expm1(k) - k)
            slope = slope - case["kl"] * torch.expm1(k)
    else:
        diff = (lp - d["ref"].double().reshape(rows)).masked_fill(dead, 0.0).reshape(shape).sum(-1)
        z = case["beta"] * (diff[:, 0] - diff[:, 1])
        eps = case["smoothing"]
        logsig = torch.nn.functional.logsigmoid
        y = -(1.0 - eps) * logsig(z) - eps * logsig(-z)
        dz = case["beta"] * (eps * torch.sigmoid(z) - (1.0 - eps) * torch.sigmoid(-z))
        slope = torch.stack([dz, -dz], 1).unsqueeze(-1).expand(shape).reshape(rows)
    if case["op"] != "preference":
        y = y.masked_fill(dead, 0.0).reshape(shape)
    if "seed" not in d:
        return [y]
    w = d["seed"].double()
    w = w[:, None, None].expand(shape).reshape(rows) if case["op"] == "preference" else w.reshape(rows)
    grad = torch.zeros(rows, V, dtype=torch.float64, device="cuda")
    for part in live.split(512):
        c = (w * slope)[part].unsqueeze(-1)
        p = -c * torch.softmax(logits[part].double(), -1)
        p[torch.arange(len(part), device="cuda"), tokens[part]] += c.squeeze(-1)
        grad[part] = p
    return [y, grad.reshape(*shape, V)]


# ---- what a case cannot do without -------------------------------------------------------------


def work(case):
    if case["op"] == "scan":
        lanes = case["B"] * case["D"]
        n = lanes * case["T"]
        gates = case["B"] * case["T"] * case["heads"] if case["heads"] else n
        init = lanes if case["init"] else 0
        if not case["train"]:  # gates, x, the first states in; the states and the last ones out
            return {"bytes": 4 * (gates + 2 * n + init + lanes), "flops": 2 * n}
        # gates, x, dh, the first states in; the states and the gradients of all inputs out
        return {"bytes": 4 * (2 * gates + 4 * n + 2 * init), "flops": 5 * n}
    rows = int(np.prod(_rows_shape(case)))
    live = int(_valid(case).sum())
    # the rows that count are read, the gradient is written in full, and some numbers a token
    small = {"logprob": 3, "policy": 5, "preference": 3}[case["op"]]
    grad = case["op"] != "logprob" or case["train"]
    return {"bytes": 4 * (case["V"] * (live + (rows if grad else 0)) + small * rows),
            "flops": case["V"] * live * (6 if grad else 4)}
