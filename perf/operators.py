"""Cases and plain forms of the operators on packed and prefix-sharing batches.

Three operators are measured:

* attention over sequences packed along one token axis, grouped heads, causal
  or not, forward alone (prompts) or with its gradient (training);
* attention of a batch whose sequences share one prefix: the prefix's keys and
  values are held once for all rows, for single tokens and for prompts;
* the norm of every query and key head with the position rotation in the same
  pass, with its gradient, and its form for single tokens that appends to the
  cache.

``own`` false: elementary torch operations in 32 bits, rounded once at the end.
``own`` true: the calls a user makes of ``kgwe.ops``.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
THETA = 500000.0


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # A few short chat turns admitted at once by a server of a small model: latency.
        {"name": "prompt_short", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 64,
         "n": 4, "lo": 1, "hi": 61, "pick": 3, "pad": 0, "causal": True, "prefix": 0, "grad": False},
        # A burst of prompts of different lengths that share one prefill pass.
        {"name": "prompt_burst", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 64,
         "n": 32, "lo": 16, "hi": 1024, "pick": 1, "pad": 0, "causal": True, "prefix": 0, "grad": False},
        # Three long documents in the other half-precision type, many query heads for each key head.
        {"name": "prompt_long", "op": "prompt", "dtype": "fp16", "hq": 16, "hkv": 2, "d": 128,
         "n": 3, "lo": 5000, "hi": 12001, "pick": 7, "pad": 0, "causal": True, "prefix": 0, "grad": False},
        # Training on packed documents at the 8B model's heads; the batch's last rows are padding.
        {"name": "train_docs", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "n": 24, "lo": 64, "hi": 4096, "pick": 2, "pad": 77, "causal": True, "prefix": 0, "grad": True},
        # Training on one long document: the largest case.
        {"name": "train_long", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "n": 1, "lo": 16384, "hi": 16384, "pick": 0, "pad": 0, "causal": True, "prefix": 0, "grad": True},
        # Questions behind one system prompt: the prompts attend to the prefix and to themselves.
        {"name": "prompt_prefix", "op": "prompt", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 64,
         "n": 16, "lo": 20, "hi": 300, "pick": 5, "pad": 0, "causal": True, "prefix": 1000, "grad": False},
        # One decode step of a small share group behind a short system prompt: latency.
        {"name": "token_prefix_small", "op": "token", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 64,
         "n": 4, "prefix": 200, "smax": 128, "lo": 0, "hi": 60, "pick": 1},
        # One decode step of a full share group (8 clients x 4 rows) behind a system prompt.
        {"name": "token_prefix_server", "op": "token", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 64,
         "n": 32, "prefix": 2048, "smax": 1024, "lo": 1, "hi": 1000, "pick": 2},
        # Many questions about one long document at the 8B model's heads.
        {"name": "token_prefix_long", "op": "token", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "n": 64, "prefix": 32768, "smax": 2048, "lo": 1, "hi": 1500, "pick": 3},
        # The new tokens of a decode step: norms, rotation and the append to the cache.
        {"name": "norm_rope_token", "op": "append", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "n": 4, "smax": 1024, "norm": True, "pick": 1},
        # A packed prefill pass of a model with small heads and no norms: the rotation alone.
        {"name": "rope_prompt", "op": "norm_rope", "dtype": "fp16", "hq": 16, "hkv": 8, "d": 64,
         "n": 9, "lo": 20, "hi": 500, "pick": 4, "pad": 3, "norm": False, "grad": False},
        # Training on packed documents: norms and rotation with their gradients.
        {"name": "norm_rope_train", "op": "norm_rope", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "n": 24, "lo": 64, "hi": 2048, "pick": 2, "pad": 5, "norm": True, "grad": True},
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "token", "token", "append", "norm_rope", "norm_rope"])
    heads = rng.choice([(32, 8), (32, 8), (16, 2), (8, 8), (12, 4), (16, 8), (5, 5), (28, 4)])
    case = {"dtype": rng.choice(["bf16", "bf16", "fp16"]), "hq": heads[0], "hkv": heads[1],
            "d": rng.choice([64, 128]), "pick": rng.randrange(1 << 20)}
    if op in ("prompt", "train"):
        n = _log_int(rng, 1, 48)
        hi = _log_int(rng, 1, min(12000, 24000 // n))
        lo = max(1, _log_int(rng, 1, hi) if n > 1 else hi)
        grad = op == "train"
        case.update(op="prompt", n=n, lo=lo, hi=hi, pad=rng.choice([0, 0, 1, 100]),
                    causal=rng.random() < 0.8, grad=grad,
                    prefix=0 if grad or rng.random() < 0.6 else _log_int(rng, 1, 4000))
    elif op == "token":
        case["hq"], case["hkv"] = rng.choice([(32, 8), (32, 8), (16, 2), (8, 8), (12, 4), (16, 8), (5, 5), (28, 4)])
        smax = _log_int(rng, 16, 4000)
        n = _log_int(rng, 1, 64)
        case.update(op="token", n=n, prefix=_log_int(rng, 1, 32768), smax=smax, lo=0,
                    hi=max(1, int(smax * rng.uniform(0.1, 1.0))))
    elif op == "append":
        case.update(op="append", n=_log_int(rng, 1, 256), smax=_log_int(rng, 16, 1500), norm=rng.random() < 0.7)
    else:
        n = _log_int(rng, 1, 48)
        hi = _log_int(rng, 1, 16000 // n)
        case.update(op="norm_rope", n=n, lo=max(1, _log_int(rng, 1, hi)), hi=hi, pad=rng.choice([0, 0, 1, 50]),
                    norm=rng.random() < 0.7, grad=rng.random() < 0.5)
    return case


def _lengths(case):
    """The sequences' lengths, spread over the logarithm of the case's range."""
    rng = random.Random(1000003 * case["pick"] + case["n"])
    lo, hi = max(case["lo"], 1), max(case["hi"], 1)
    out = [_log_int(rng, lo, hi) for _ in range(case["n"])]
    if case["lo"] == 0 and case["n"] > 1:  # a row with nothing of its own yet
        out[rng.randrange(case["n"])] = 0
    return out


def _rows(case):
    return sum(_lengths(case)) + case.get("pad", 0)


def work(case):
    es = 2
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "prompt":
        lens, T, P = _lengths(case), _rows(case), case["prefix"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens) + P * sum(lens)
        rd = (T * hq + 2 * T * hkv + 2 * P * hkv) * d * es
        wr = T * hq * d * es
        flops = 4 * d * hq * pairs
        if case["grad"]:
            rd += T * hq * d * es
            wr += (T * hq + 2 * T * hkv) * d * es
            flops += 10 * d * hq * pairs
        return {"bytes": rd + wr + 4 * (case["n"] + 1), "flops": flops}
    if case["op"] == "token":
        keys = sum(_lengths(case))
        n, P = case["n"], case["prefix"]
        return {"bytes": 2 * n * hq * d * es + 2 * hkv * d * es * (P + keys) + 4 * n,
                "flops": 4 * d * hq * (n * P + keys)}
    rows = case["n"] if case["op"] == "append" else _rows(case)
    width = (hq + 2 * hkv) * d
    table = min(rows, case["smax"] if case["op"] == "append" else max(_lengths(case))) * d * 4
    b, f = 2 * rows * width * es + 4 * rows + table, 8 * rows * (hq + hkv) * d
    if case.get("grad"):
        b += 2 * rows * width * es
        f += 16 * rows * (hq + hkv) * d
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ the inputs
def _inputs(case, seed):
    dev = torch.device("cuda")
    dt = DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]

    def rnd(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=g).mul_(scale).to(dt)

    x = {}
    if case["op"] == "prompt":
        T, P = _rows(case), case["prefix"]
        # Queries with some sharp heads, as trained models have them.
        x["q"] = (rnd(T, hq, d) * torch.linspace(0.5, 2.0, hq, device=dev).to(dt)[None, :, None]).contiguous()
        x["k"], x["v"] = rnd(T, hkv, d), rnd(T, hkv, d)
        if P:
            x["pk"], x["pv"] = rnd(hkv, P, d), rnd(hkv, P, d)
        if case["grad"]:
            x["do"] = rnd(T, hq, d, scale=0.5)
    elif case["op"] == "token":
        n, P, smax = case["n"], case["prefix"], case["smax"]
        x["q"] = (rnd(n, hq, d) * torch.linspace(0.5, 2.0, hq, device=dev).to(dt)[None, :, None]).contiguous()
        x["pk"], x["pv"] = rnd(hkv, P, d), rnd(hkv, P, d)
        x["kc"], x["vc"] = rnd(n, hkv, smax, d), rnd(n, hkv, smax, d)  # past its length a row holds stale keys
        x["lens"] = torch.tensor([min(m, smax) for m in _lengths(case)], dtype=torch.int32, device=dev)
    else:
        append = case["op"] == "append"
        rows = case["n"] if append else _rows(case)
        x["qkv"] = rnd(rows, (hq + 2 * hkv) * d, scale=1.5)
        if case["norm"]:
            x["wq"] = (1 + 0.2 * torch.randn(d, device=dev, generator=g)).to(dt)
            x["wk"] = (1 + 0.2 * torch.randn(d, device=dev, generator=g)).to(dt)
        longest = case["smax"] if append else max(_lengths(case))
        angle = (torch.arange(longest, dtype=torch.float64)[:, None]
                 * THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)[None, :])
        x["cos"], x["sin"] = angle.cos().float().to(dev), angle.sin().float().to(dev)
        if append:
            x["pos"] = torch.randint(0, case["smax"], (rows,), device=dev, generator=g, dtype=torch.int32)
            x["kc"], x["vc"] = rnd(rows, hkv, case["smax"], d), rnd(rows, hkv, case["smax"], d)
        else:
            x["pos"] = torch.cat([torch.arange(m, dtype=torch.int32) for m in _lengths(case)]
                                 + [torch.full((case["pad"],), -1, dtype=torch.int32)]).to(dev)
            if case["grad"]:
                x["dq"], x["dk"], x["dv"] = rnd(rows, hq, d), rnd(rows, hkv, d), rnd(rows, hkv, d)
    return x


def prepare(case, seed):
    state = {"case": case, "x": _inputs(case, seed)}
    x = state["x"]
    if case["op"] == "prompt":
        state["lens"] = _lengths(case)
    if own:
        from kgwe.ops import decode, packed
        if case["op"] == "prompt":
            state["batch"] = packed.PackedBatch(state["lens"], total=x["q"].shape[0], device=x["q"].device)
            if case["grad"]:
                for name in ("q", "k", "v"):
                    x[name].requires_grad_(True)
        elif case["op"] == "token":
            state["attend"] = decode.PrefixDecodeAttention(case["n"], case["hq"], case["hkv"], case["d"],
                                                           case["smax"], case["prefix"], x["q"].device,
                                                           dtype=x["q"].dtype)
        elif case.get("grad"):
            for name in ("qkv", "wq", "wk"):
                if name in x:
                    x[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------ the calls
def run(state):
    case, x = state["case"], state["x"]
    return (_run_own if own else _run_plain)[case["op"]](case, x, state)


def _own_prompt(case, x, state):
    from kgwe.ops import attn
    if case["prefix"]:
        return attn.attention_packed(x["q"], x["k"], x["v"], state["batch"], causal=case["causal"],
                                     prefix=(x["pk"], x["pv"]))
    o = attn.attention_packed(x["q"], x["k"], x["v"], state["batch"], causal=case["causal"])
    if not case["grad"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, (x["q"], x["k"], x["v"]), x["do"]))


def _own_token(case, x, state):
    return state["attend"](x["q"], x["pk"], x["pv"], x["kc"], x["vc"], x["lens"])


def _own_append(case, x, state):
    from kgwe.ops import decode
    q = decode.norm_rope_append(x["qkv"], x["pos"], x["cos"], x["sin"], x["kc"], x["vc"], case["hq"], case["hkv"],
                                case["d"], q_weight=x.get("wq"), k_weight=x.get("wk"), eps=EPS)
    return q, x["kc"], x["vc"]


def _own_norm_rope(case, x, state):
    from kgwe.ops import functional
    out = functional.norm_rope_qkv(x["qkv"], x["cos"], x["sin"], x["pos"], case["hq"], case["hkv"], case["d"],
                                   q_weight=x.get("wq"), k_weight=x.get("wk"), eps=EPS)
    if not case["grad"]:
        return out
    leaves = [x[name] for name in ("qkv", "wq", "wk") if name in x]
    grads = torch.autograd.grad(out, leaves, (x["dq"], x["dk"], x["dv"]))
    return (*(t.detach() for t in out), *grads)


_run_own = {"prompt": _own_prompt, "token": _own_token, "append": _own_append, "norm_rope": _own_norm_rope}


# ------------------------------------------------------------------ the plain forms
def _grouped(t, hkv):
    """[L, H, D] -> fp32 [Hkv, G * L, D] (the heads of a group one after the other)."""
    L, H, D = t.shape
    return t.float().view(L, hkv, H // hkv, D).permute(1, 2, 0, 3).reshape(hkv, H // hkv * L, D)


def _ungrouped(t, L):
    """[Hkv, G * L, D] -> [L, H, D]."""
    hkv, GL, D = t.shape
    return t.view(hkv, GL // L, L, D).permute(2, 0, 1, 3).reshape(L, hkv * (GL // L), D)


def _plain_prompt(case, x, state):
    hkv, d = case["hkv"], case["d"]
    G, scale = case["hq"] // hkv, 1.0 / math.sqrt(d)
    dt = x["q"].dtype
    names = ("q", "k", "v") if case["grad"] else ()
    o = torch.zeros_like(x["q"])
    grads = {name: torch.zeros_like(x[name]) for name in names}
    P = case["prefix"]
    at = 0
    for L in state["lens"]:
        if L == 0:
            continue
        rows = slice(at, at + L)
        at += L
        k, v = (x[name][rows].float().transpose(0, 1) for name in ("k", "v"))  # [Hkv, L, D]
        if P:
            k, v = torch.cat([x["pk"].float(), k], 1), torch.cat([x["pv"].float(), v], 1)
        q = _grouped(x["q"][rows], hkv)
        do = _grouped(x["do"][rows], hkv) if case["grad"] else None
        hidden = None
        if case["causal"]:
            hidden = torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1)
            hidden = torch.nn.functional.pad(hidden, (P, 0)).repeat(G, 1)
        # One key head at a time where the scores of all of them would be many gigabytes.
        step = max(1, min(hkv, (1 << 30) // max(1, G * L * (L + P))))
        oh = torch.empty_like(q)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        for h in range(0, hkv, step):
            hs = slice(h, h + step)
            s = torch.matmul(q[hs], k[hs].transpose(1, 2)).mul_(scale)
            if hidden is not None:
                s.masked_fill_(hidden, float("-inf"))
            p = s.sub_(s.amax(-1, keepdim=True)).exp_()
            p /= p.sum(-1, keepdim=True)
            oh[hs] = torch.matmul(p, v[hs])
            if case["grad"]:
                dv[hs] = torch.matmul(p.transpose(1, 2), do[hs])
                ds = torch.matmul(do[hs], v[hs].transpose(1, 2))
                ds -= (do[hs] * oh[hs]).sum(-1, keepdim=True)
                ds.mul_(p).mul_(scale)
                dq[hs] = torch.matmul(ds, k[hs])
                dk[hs] = torch.matmul(ds.transpose(1, 2), q[hs])
        o[rows] = _ungrouped(oh, L).to(dt)
        if case["grad"]:
            grads["q"][rows] = _ungrouped(dq, L).to(dt)
            grads["k"][rows] = dk.transpose(0, 1).to(dt)
            grads["v"][rows] = dv.transpose(0, 1).to(dt)
    return (o, *(grads[name] for name in names)) if names else o


def _plain_token(case, x, state):
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    G, smax = hq // hkv, case["smax"]
    q = x["q"].float().view(n, hkv, G, d) / math.sqrt(d)
    qh = q.permute(1, 0, 2, 3).reshape(hkv, n * G, d)
    sp = torch.matmul(qh, x["pk"].float().transpose(1, 2)).view(hkv, n, G, -1).permute(1, 0, 2, 3)
    so = torch.matmul(q, x["kc"].float().transpose(2, 3))
    hidden = torch.arange(smax, device=q.device)[None, :] >= x["lens"][:, None]
    so = so.masked_fill(hidden[:, None, None, :], float("-inf"))
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    pp, po = torch.exp(sp - m), torch.exp(so - m)
    total = pp.sum(-1, keepdim=True) + po.sum(-1, keepdim=True)
    op = torch.matmul(pp.permute(1, 0, 2, 3).reshape(hkv, n * G, -1), x["pv"].float())
    op = op.view(hkv, n, G, d).permute(1, 0, 2, 3)
    return ((op + torch.matmul(po, x["vc"].float())) / total).reshape(n, hq, d).to(x["q"].dtype)


def _rotate(t, c, s):
    a, b = t.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _norm_rotate(h, w, c, s):
    if w is not None:
        h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * w.float()
    return _rotate(h, c, s)


def _norm_rotate_grad(dy, h, w, c, s):
    """Gradients of _norm_rotate with regard to h and w."""
    g = _rotate(dy, c, -s)
    if w is None:
        return g, None
    r = torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + EPS)
    gw = g * w.float()
    dx = r * (gw - h * r * r * (gw * h).mean(-1, keepdim=True))
    return dx, (g * h * r).sum((0, 1))


def _plain_append(case, x, state):
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    dt = x["qkv"].dtype
    h = x["qkv"].float().view(n, hq + 2 * hkv, d)
    pos = x["pos"].long()
    c, s = x["cos"][pos][:, None], x["sin"][pos][:, None]
    row = torch.arange(n, device=pos.device)
    x["kc"][row, :, pos] = _norm_rotate(h[:, hq:hq + hkv], x.get("wk"), c, s).to(dt)
    x["vc"][row, :, pos] = h[:, hq + hkv:].to(dt)
    return _norm_rotate(h[:, :hq], x.get("wq"), c, s).to(dt), x["kc"], x["vc"]


def _plain_norm_rope(case, x, state):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    dt = x["qkv"].dtype
    h = x["qkv"].float().view(-1, hq + 2 * hkv, d)
    live = (x["pos"] >= 0)[:, None, None]  # a row without a position is padding: zero, and so is its gradient
    pos = x["pos"].clamp(min=0).long()
    c, s = x["cos"][pos][:, None], x["sin"][pos][:, None]
    parts = (h[:, :hq], h[:, hq:hq + hkv], h[:, hq + hkv:])
    wq, wk = x.get("wq"), x.get("wk")
    out = (_norm_rotate(parts[0], wq, c, s), _norm_rotate(parts[1], wk, c, s), parts[2])
    out = tuple((t * live).to(dt) for t in out)
    if not case["grad"]:
        return out
    gq, dwq = _norm_rotate_grad(x["dq"].float() * live, parts[0], wq, c, s)
    gk, dwk = _norm_rotate_grad(x["dk"].float() * live, parts[1], wk, c, s)
    dqkv = torch.cat([gq, gk, x["dv"].float() * live], dim=1).reshape(x["qkv"].shape).to(dt)
    return (*out, dqkv, *(t.to(dt) for t in (dwq, dwk) if t is not None))


_run_plain = {"prompt": _plain_prompt, "token": _plain_token, "append": _plain_append,
              "norm_rope": _plain_norm_rope}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    x = {name: t.double() if t.is_floating_point() else t for name, t in _inputs(case, seed).items()}
    return {"prompt": _exact_prompt, "token": _exact_token, "append": _exact_append,
            "norm_rope": _exact_norm_rope}[case["op"]](case, x)


def _exact_prompt(case, x):
    G, root = case["hq"] // case["hkv"], math.sqrt(case["d"])
    o = torch.zeros_like(x["q"])
    dq, dk, dv = (torch.zeros_like(x[name]) for name in ("q", "k", "v"))
    start = 0
    for L in _lengths(case):
        end = start + L
        i = torch.arange(L, device=o.device)
        for h in range(case["hq"]):
            j = h // G
            keys, vals = x["k"][start:end, j], x["v"][start:end, j]
            seen = (i[:, None] >= i[None, :]) if case["causal"] else torch.ones(L, L, dtype=torch.bool,
                                                                                device=o.device)
            if case["prefix"]:
                keys, vals = torch.cat((x["pk"][j], keys)), torch.cat((x["pv"][j], vals))
                seen = torch.cat((seen.new_ones(L, case["prefix"]), seen), 1)
            logit = torch.where(seen, x["q"][start:end, h] @ keys.T / root, -math.inf)
            p = torch.softmax(logit, dim=1)
            o[start:end, h] = p @ vals
            if case["grad"]:
                up = x["do"][start:end, h]
                dp = up @ vals.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / root
                dq[start:end, h] = ds @ keys
                dk[start:end, j] += ds.T @ x["q"][start:end, h]
                dv[start:end, j] += p.T @ up
        start = end
    return (o, dq, dk, dv) if case["grad"] else o


def _exact_token(case, x):
    G, root = case["hq"] // case["hkv"], math.sqrt(case["d"])
    out = torch.zeros_like(x["q"])
    for b, L in enumerate(x["lens"].tolist()):
        for j in range(case["hkv"]):
            keys = torch.cat((x["pk"][j], x["kc"][b, j, :L]))
            vals = torch.cat((x["pv"][j], x["vc"][b, j, :L]))
            hs = slice(j * G, (j + 1) * G)
            out[b, hs] = torch.softmax(x["q"][b, hs] @ keys.T / root, dim=1) @ vals
    return out


def _turned(case, x, first, heads, w):
    """Norm and rotation of `heads` heads from head `first` on, as complex numbers; differentiable."""
    d = case["d"]
    h = x["qkv"].reshape(len(x["pos"]), -1, d)[:, first:first + heads]
    if w is not None:
        h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / d + EPS) * w
    z = torch.complex(h[..., :d // 2], h[..., d // 2:])
    at = x["pos"].clamp(min=0).long()
    z = z * torch.complex(x["cos"][at], x["sin"][at])[:, None]
    return torch.cat((z.real, z.imag), -1) * (x["pos"] >= 0)[:, None, None]


def _exact_append(case, x):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    k = _turned(case, x, hq, hkv, x.get("wk"))
    v = x["qkv"].reshape(case["n"], -1, d)[:, hq + hkv:]
    for b, p in enumerate(x["pos"].tolist()):
        x["kc"][b, :, p], x["vc"][b, :, p] = k[b], v[b]
    return _turned(case, x, 0, hq, x.get("wq")), x["kc"], x["vc"]


def _exact_norm_rope(case, x):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    leaves = [x[name] for name in ("qkv", "wq", "wk") if name in x]
    if case["grad"]:
        for leaf in leaves:
            leaf.requires_grad_(True)
    v = x["qkv"].reshape(len(x["pos"]), -1, d)[:, hq + hkv:] * (x["pos"] >= 0)[:, None, None]
    out = (_turned(case, x, 0, hq, x.get("wq")), _turned(case, x, hq, hkv, x.get("wk")), v)
    if not case["grad"]:
        return out
    grads = torch.autograd.grad(out, leaves, (x["dq"], x["dk"], x["dv"]))
    return (*(t.detach() for t in out), *grads)
