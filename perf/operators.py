"""Workloads of the policy operators: drawing actions from a policy, the
policy loss with its gradient, and the optimiser step.

`run` computes them in plain torch operations, or through the package's
entry points where `own` is true.  All inputs are made from a seed.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
FLT_MAX = 3.4028234663852886e38
BLOCK = 256  # elements of an 8-bit state block
BETA1, BETA2, EPS = 0.9, 0.999, 1e-8


def listed():
    """The cases.  sample: actions drawn from masked rows; loss: the policy
    loss and its gradient; adamw: one optimiser step over a model's tensors."""
    sample = dict(op="sample", pad=0, legal=0, temp=1.0, top_k=0, top_p=1.0, min_p=0.0, per_row=False)
    loss = dict(op="loss", legal=0, dense=False, weighted=False)
    adamw = dict(op="adamw", features=4, actions=7, bits=32, grad="f32", copy="", clip=0.0, lr=1e-3)
    return [
        # one move of one Connect4 game, as an interactive player asks for it
        dict(sample, name="sample_connect4_move", rows=1, actions=7, dtype="f32", legal=6),
        # a wave of 1024 chess games from the 4672-way policy, the opening at
        # temperature 1 and later moves greedy
        dict(sample, name="sample_chess_games", rows=1024, actions=4672, dtype="f32", legal=34, per_row=True),
        # 4096 chess positions with filtered sampling, in 16 bits
        dict(sample, name="sample_chess_filtered", rows=4096, actions=4672, dtype="f16", legal=34, temp=0.8, top_p=0.95,
             min_p=0.02),
        # one token over a vocabulary whose size is odd, in rows of a padded buffer
        dict(sample, name="sample_vocabulary_one", rows=1, actions=100003, dtype="bf16", pad=61, temp=0.7, top_k=50,
             top_p=0.9),
        # a serving batch over a large vocabulary, nucleus sampling
        dict(sample, name="sample_vocabulary_batch", rows=256, actions=131072, dtype="bf16", top_p=0.92),
        # the training batch of the Connect4 networks
        dict(loss, name="loss_connect4_batch", rows=64, actions=7, dtype="f32", legal=6, dense=True),
        # search policies as targets over legal chess moves
        dict(loss, name="loss_chess_targets", rows=8192, actions=4672, dtype="f32", legal=34, dense=True),
        # the actions taken, weighted by their advantages, over an odd vocabulary
        dict(loss, name="loss_vocabulary_taken", rows=2048, actions=100003, dtype="bf16", weighted=True),
        # few long rows in 32 bits
        dict(loss, name="loss_long_rows", rows=4, actions=131072, dtype="f32"),
        # the Connect4 graph-attention network's tensors, 8-bit states
        dict(adamw, name="adamw_connect4_8bit", layers=6, width=256, bits=8),
        # 50 M weights: 8-bit states, 16-bit gradients and working copy, clipping
        dict(adamw, name="adamw_wide_8bit", layers=12, width=2048, features=18, actions=4672, bits=8, grad="bf16",
             copy="bf16", clip=1.0, lr=1e-4),
        # 200 M weights: 32-bit states
        dict(adamw, name="adamw_wide_32bit", layers=12, width=4096, features=18, actions=4672, grad="bf16", copy="bf16",
             lr=1e-4),
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of lo..hi."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(hi, max(lo, n))
    return n + 1 if n == 3072 else n


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["sample", "loss", "adamw"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "adamw":
        layers, width = rng.randint(1, 12), _between(rng, 16, 2048)
        return dict(op=op, layers=layers, width=width, features=rng.choice([2, 4, 18]), actions=rng.choice([7, 9, 4672]),
                    bits=rng.choice([8, 32]), grad=rng.choice(["f32", "f16", "bf16"]), copy=rng.choice(["", "f16", "bf16"]),
                    clip=rng.choice([0.0, 1.0]), lr=1e-4)
    actions = rng.choice([7, 9, 4672, _between(rng, 2, 131072), _between(rng, 2, 131072)])
    if op == "loss":
        rows = _between(rng, 1, min(8192, max(1, 32000000 // actions)))
        legal = rng.choice([0, max(1, min(34, actions - 1))])
        return dict(op=op, rows=rows, actions=actions, dtype=dtype, legal=legal, dense=rng.random() < 0.5,
                    weighted=rng.random() < 0.5)
    rows = _between(rng, 1, min(4096, max(1, 33554432 // actions)))
    legal = rng.choice([0, max(1, min(34, actions - 1))])
    return dict(op=op, rows=rows, actions=actions, dtype=dtype, pad=rng.choice([0, 0, 1, 13]), legal=legal,
                temp=rng.choice([0.6, 1.0, 1.3]), top_k=rng.choice([0, 0, _between(rng, 1, 200)]),
                top_p=rng.choice([1.0, 0.9, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, 0.0, 0.05]),
                per_row=rng.random() < 0.3)


def _shapes(case):
    """The tensors of a graph-attention network: per layer weights, bias and
    attention vectors, then the value and the policy head."""
    d, a = case["width"], case["actions"]
    shapes = []
    for k in range(case["layers"]):
        shapes += [(case["features"] if k == 0 else d, d), (d,), (2, d)]
    return shapes + [(d, 64), (64,), (64,), (1,), (d, a), (a,)]


def _counts(case):
    n = [math.prod(s) for s in _shapes(case)]
    return n, [-(-k // BLOCK) * BLOCK for k in n]


def work(case):
    """Bytes: each input read once, each output written once; of the noise only
    what a top-k keeps, and none where the kept share depends on the data.
    Flops: about one per arithmetic operation of the formulas."""
    if case["op"] == "adamw":
        n = sum(_counts(case)[0])
        per = 8 + SIZES[case["grad"]] + (16 if case["bits"] == 32 else 4 + 16 / BLOCK) + (2 if case["copy"] else 0)
        return {"bytes": n * per, "flops": 16 * n}
    r, a, e = case["rows"], case["actions"], SIZES[case["dtype"]]
    if case["op"] == "loss":
        read = a * e + (a if case["legal"] else 0) + (4 * a if case["dense"] else 4) + (4 if case["weighted"] else 0)
        return {"bytes": r * (read + a * e + 4), "flops": r * a * 8}
    if case["top_k"]:
        noise = 4 * min(case["top_k"], a)
    elif case["top_p"] < 1 or case["min_p"] > 0 or case["legal"]:
        noise = 4
    else:
        noise = 4 * a
    return {"bytes": r * (a * e + (a if case["legal"] else 0) + noise + 8 + (16 if case["per_row"] else 0)),
            "flops": r * a * 4}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(case, g):
    """Scores as policy heads give them: a broad bell and a few high peaks."""
    r, a = case["rows"], case["actions"]
    x = torch.randn(r, a + case.get("pad", 0), generator=g, device="cuda")
    x = 2 * x + 5 * torch.relu(x - 2.5)
    return x.to(DTYPES[case["dtype"]])[:, :a]


def _mask(case, g):
    """Legal actions; about one row in a hundred belongs to a finished game."""
    if not case["legal"]:
        return None
    r, a = case["rows"], case["actions"]
    m = torch.rand(r, a, generator=g, device="cuda") < case["legal"] / a
    if r > 1:
        m[torch.rand(r, generator=g, device="cuda") < 0.01] = False
    else:
        m[0, a // 2] = True
    return m.to(torch.uint8)


def _prepare_adamw(case, g):
    n, padded = _counts(case)
    total = sum(padded)
    at, views = 0, []
    for s, k, p in zip(_shapes(case), n, padded):
        views.append((at, k, s))
        at += p
    used = torch.zeros(total, device="cuda")
    for at, k, s in views:
        used[at:at + k] = 1
    param = 0.02 * torch.randn(total, generator=g, device="cuda") * used
    size = torch.exp(torch.randn(total, generator=g, device="cuda")) * 1e-3
    grad = (size * torch.randn(total, generator=g, device="cuda") * used).to(DTYPES[case["grad"]])
    m = 0.3 * size * torch.randn(total, generator=g, device="cuda") * used
    v = size * size * (0.5 + torch.rand(total, generator=g, device="cuda")) * used
    cut = lambda t: [t[at:at + k].view(s) for at, k, s in views]  # noqa: E731
    copy = param.to(DTYPES[case["copy"]]) if case["copy"] else None
    state = dict(case=case, param=param, grad=grad, grads=cut(grad), copy=copy, step=200)
    if case["bits"] == 32:
        state |= dict(m=m, v=v, m_scale=None, v_scale=None)
    else:
        key = torch.arange(total, device="cuda") * 40503 & 0xFFFFFFFF
        state["m"], state["m_scale"] = _to_8bit(m, (key & 0xFFFF).float() * 2.0**-16, False)
        state["v"], state["v_scale"] = _to_8bit(torch.sqrt(v), (key >> 16).float() * 2.0**-16, True)
    if own:
        import graphzero_b200 as gz

        opt = gz.AdamW(cut(param), lr=case["lr"], betas=(BETA1, BETA2), eps=EPS, weight_decay=0.01,
                       state_bits=case["bits"], copies=cut(copy) if case["copy"] else None, max_norm=case["clip"], seed=7)
        opt.steps = state["step"]
        opt.m.copy_(state["m"])
        opt.v.copy_(state["v"])
        if case["bits"] == 8:
            opt.m_scale.copy_(state["m_scale"])
            opt.v_scale.copy_(state["v_scale"])
        state |= dict(opt=opt, m=opt.m, v=opt.v, m_scale=opt.m_scale, v_scale=opt.v_scale)
    return state


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, g)
    r, a = case["rows"], case["actions"]
    state = dict(case=case, logits=_logits(case, g), mask=_mask(case, g))
    if case["op"] == "sample":
        state["noise"] = -torch.empty(r, a, device="cuda").exponential_(generator=g).log()
        for key, name, kind in (("temperature", "temp", torch.float32), ("top_k", "top_k", torch.int32),
                                ("top_p", "top_p", torch.float32), ("min_p", "min_p", torch.float32)):
            state[key] = torch.full((r,), case[name], dtype=kind, device="cuda") if case["per_row"] else case[name]
        if case["per_row"]:  # half of the games are past their opening: greedy
            state["temperature"][torch.rand(r, generator=g, device="cuda") < 0.5] = 0
        return state
    state |= dict(target=None, label=None, weight=None)
    if case["dense"]:  # visit shares: a few actions of each row, most of the legal ones at zero
        t = torch.rand(r, a, generator=g, device="cuda") ** 8
        if state["mask"] is not None:
            t = t * state["mask"]
        state["target"] = t / t.sum(1, keepdim=True).clamp(min=1e-9)
    else:
        pick = torch.rand(r, a, generator=g, device="cuda")
        if state["mask"] is not None:
            pick = pick * state["mask"]
        state["label"] = pick.argmax(1).to(torch.int32)
    if case["weighted"]:
        state["weight"] = torch.randn(r, generator=g, device="cuda")
    return state


# ---- plain forms ------------------------------------------------------------


def _column(x, like, kind):
    """A setting as a column: one value for every row, or a tensor's."""
    if isinstance(x, torch.Tensor):
        return x[:, None]
    return torch.full((1, 1), x, dtype=kind, device=like.device)


def _sample_plain(s):
    x = s["logits"].float()
    ninf = torch.full((), -math.inf, device=x.device)
    seen = x > -math.inf  # false for NaN
    if s["mask"] is not None:
        seen = seen & (s["mask"] != 0)
    x = torch.where(seen, x.clamp(max=FLT_MAX), ninf)
    top, first = x.max(1, keepdim=True)[0], x.argmax(1, keepdim=True)
    some = top > -math.inf
    t = _column(s["temperature"], x, torch.float32)
    greedy = ~(t > 0)
    d = (x - torch.where(some, top, torch.zeros_like(top))) / torch.where(greedy, torch.ones_like(t), t)
    e = torch.exp(d)
    top_k, top_p, min_p = (_column(s[k], x, kind) for k, kind in
                           (("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)))
    case = s["case"]
    keep = seen
    if case["top_k"] or case["top_p"] < 1:
        order = torch.sort(x, dim=1, descending=True, stable=True)[1]
        rank = torch.arange(x.shape[1], device=x.device)[None, :]
        weight = torch.gather(e, 1, order)
        weight = torch.where((top_k <= 0) | (rank < top_k), weight, torch.zeros_like(weight))
        before = torch.cumsum(weight, 1) - weight
        chosen = ((top_k <= 0) | (rank < top_k)) & ((top_p >= 1) | (rank == 0) | (before < top_p * weight.sum(1, keepdim=True)))
        keep = seen & torch.zeros_like(seen).scatter(1, order, chosen)
    keep = keep & (e >= min_p)
    keep = torch.where(greedy, torch.arange(x.shape[1], device=x.device)[None, :] == first, keep) & seen
    action = torch.where(keep, d + s["noise"], ninf).argmax(1, keepdim=True)
    z = torch.where(keep, e, torch.zeros_like(e)).sum(1, keepdim=True)
    logp = torch.gather(d, 1, action) - torch.log(z)
    logp = torch.where(some, logp, torch.zeros_like(logp))
    action = torch.where(some, action, torch.full_like(action, -1))
    return {"action": action[:, 0].to(torch.int32), "logp": logp[:, 0]}


def _loss_plain(s):
    x = s["logits"].float()
    seen = torch.ones_like(x, dtype=torch.bool) if s["mask"] is None else s["mask"] != 0
    x = torch.where(seen, x, torch.full((), -math.inf, device=x.device))
    top = x.amax(1, keepdim=True)
    live = top != -math.inf
    d = x - torch.where(live, top, torch.zeros_like(top))
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    if s["target"] is not None:
        t = torch.where(seen & live, s["target"], torch.zeros_like(x))
    else:
        at = s["label"].long()[:, None]
        t = (torch.arange(x.shape[1], device=x.device)[None, :] == at) & seen & live
        t = t.float()
    mass = t.sum(1, keepdim=True)
    cross = torch.where(t != 0, t * d, torch.zeros_like(d)).sum(1, keepdim=True)
    w = torch.ones_like(mass) if s["weight"] is None else s["weight"][:, None]
    scale = 1.0 / x.shape[0]
    loss = torch.where(live, w * (mass * torch.log(z) - cross), torch.zeros_like(mass))
    share = torch.where(live, mass / z, torch.zeros_like(mass))
    grad = (w * scale) * (e * share - t)
    return {"loss": loss[:, 0], "grad": grad.to(s["logits"].dtype)}


def _power(exponent):
    """2 to the exponent, as 32-bit floats (exponent: int32, -126..127)."""
    return ((exponent + 127) << 23).view(torch.float32)


def _mix32(x):
    """The 32-bit integer hash that the package rounds weights by (int64 tensors)."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _to_8bit(x, u, nonzero):
    """Blocks of 256 as 8-bit floats (4 exponent bits, 3 mantissa bits) and a
    power-of-two scale that brings the block's largest to 448 at most; rounded
    down or up by u in [0, 1).  nonzero: a positive value stays above zero."""
    y = x.view(-1, BLOCK)
    bits = y.abs().amax(1, keepdim=True).view(torch.int32)
    k = (bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)
    k = torch.where(bits == 0, torch.zeros_like(k), k.clamp(min=-126))
    y = y.abs() * _power(-k)
    e = ((y.view(torch.int32) >> 23) - 127).clamp(min=-6)
    q = torch.floor(y * _power(3 - e) + u.view(-1, BLOCK))
    if nonzero:
        q = torch.where((q == 0) & (y > 0), torch.ones_like(q), q)
    q = torch.copysign(q * _power(e - 3), x.view(-1, BLOCK))
    return q.view(-1).to(torch.float8_e4m3fn), _power(k).view(-1)


def _from_8bit(q, scale):
    return (q.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _adamw_settings(s):
    """Step size, decay factor and the second moment's correction, in doubles."""
    lr, step = s["case"]["lr"], s["step"]
    return lr / (1 - BETA1**step), 1 - lr * 0.01, 1 / math.sqrt(1 - BETA2**step)


def _rounding(s, n, device):
    """The step's rounding numbers in [0, 1) for the two states."""
    key = _mix32(torch.tensor((s["step"] * 0x9E3779B9 + 7) & 0xFFFFFFFF, device=device))
    h = _mix32((torch.arange(n, device=device) + key) & 0xFFFFFFFF)
    return (h & 0xFFFF).float() * 2.0**-16, (h >> 16).float() * 2.0**-16


def _adamw_plain(s):
    s["step"] += 1
    case, p = s["case"], s["param"]
    step, decay, correct = _adamw_settings(s)
    g = s["grad"].float()
    norm = None
    if case["clip"]:
        norm = torch.sqrt((g * g).sum())
        g = g * torch.clamp(case["clip"] / (norm + 1e-6), max=1.0)
    if case["bits"] == 8:
        m, r = _from_8bit(s["m"], s["m_scale"]), _from_8bit(s["v"], s["v_scale"])
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    root = torch.sqrt(v)
    p.copy_(p * decay - m / (root * correct + EPS) * step)
    if case["bits"] == 8:
        um, uv = _rounding(s, p.numel(), p.device)
        s["m"], s["m_scale"] = _to_8bit(m, um, False)
        s["v"], s["v_scale"] = _to_8bit(root, uv, True)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if case["copy"]:
        s["copy"].copy_(p)
    return _adamw_outputs(s, norm)


def _adamw_outputs(s, norm):
    return {k: x for k, x in dict(param=s["param"], m=s["m"], v=s["v"], m_scale=s["m_scale"], v_scale=s["v_scale"],
                                  copy=s["copy"], norm=norm).items() if x is not None}


def run(state):
    s, case = state, state["case"]
    if own:
        import graphzero_b200 as gz

        if case["op"] == "sample":
            action, logp = gz.policy_sample(s["logits"], s["noise"], mask=s["mask"], temperature=s["temperature"],
                                            top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
            return {"action": action, "logp": logp}
        if case["op"] == "loss":
            loss, grad = gz.policy_loss(s["logits"], target=s["target"], label=s["label"], mask=s["mask"],
                                        weight=s["weight"], grad_scale=1.0 / case["rows"])
            return {"loss": loss, "grad": grad}
        return _adamw_outputs(s, s["opt"].step(s["grads"]))
    return {"sample": _sample_plain, "loss": _loss_plain, "adamw": _adamw_plain}[case["op"]](s)


# ---- the definitions in 64 bits ----------------------------------------------


def _exact_sample(s):
    """Row by row: sort the visible actions, walk down the list."""
    case = s["case"]
    value = lambda k: s[k].double().tolist() if case["per_row"] else [float(case[{"temperature": "temp"}.get(k, k)])] * case["rows"]  # noqa: E731
    temperature, top_k, top_p, min_p = (value(k) for k in ("temperature", "top_k", "top_p", "min_p"))
    x, noise = s["logits"].double().cpu(), s["noise"].double().cpu()
    mask = None if s["mask"] is None else s["mask"].cpu()
    actions, logps = [], []
    for i in range(case["rows"]):
        seen = torch.arange(case["actions"]) if mask is None else mask[i].nonzero()[:, 0]
        if not len(seen):
            actions.append(-1)
            logps.append(0.0)
            continue
        row = x[i, seen]
        place = torch.sort(-row, stable=True)[1]
        seen, row = seen[place], row[place]
        if temperature[i] <= 0:
            actions.append(int(seen[0]))
            logps.append(0.0)
            continue
        if top_k[i] > 0:
            seen, row = seen[:int(top_k[i])], row[:int(top_k[i])]
        d = (row - row[0]) / temperature[i]
        p = d.exp() / d.exp().sum()
        if top_p[i] < 1:
            n = max(1, int((p.cumsum(0) - p < top_p[i]).sum()))
            seen, d, p = seen[:n], d[:n], p[:n]
        n = max(1, int((d.exp() >= min_p[i]).sum()))
        seen, d = seen[:n], d[:n]
        at = int((d + noise[i, seen]).argmax())
        actions.append(int(seen[at]))
        logps.append(float(d[at] - d.exp().sum().log()))
    return {"action": torch.tensor(actions, dtype=torch.int32), "logp": torch.tensor(logps, dtype=torch.float64)}


def _exact_loss(s):
    """In slices of rows: log-probabilities by logsumexp, and the definition of the gradient."""
    case, losses, grads = s["case"], [], []
    rows = max(1, (1 << 25) // case["actions"])
    for at in range(0, case["rows"], rows):
        to = slice(at, at + rows)
        x = s["logits"][to].double()
        if s["mask"] is not None:
            x = x.masked_fill(s["mask"][to] == 0, -math.inf)
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        dead = torch.isnan(logp).all(1, keepdim=True)
        p = torch.nan_to_num(logp.exp(), nan=0.0)
        if s["target"] is not None:
            t = s["target"][to].double()
        else:
            t = torch.zeros_like(x)
            t[torch.arange(x.shape[0], device=x.device), s["label"][to].long()] = 1
        t = t.masked_fill(torch.isinf(x) | dead, 0.0)
        w = 1.0 if s["weight"] is None else s["weight"][to].double()
        losses.append(-w * (t * logp.masked_fill(t == 0, 0.0)).sum(1))
        w = w if isinstance(w, float) else w[:, None]
        grads.append((w * (p * t.sum(1, keepdim=True) - t) / case["rows"]).cpu())
    return {"loss": torch.cat(losses), "grad": torch.cat(grads)}


def _exact_8bit(x, u, nonzero):
    y = x.view(-1, BLOCK)
    most = y.abs().amax(1, keepdim=True)
    scale = torch.where(most > 0, 2.0 ** torch.ceil(torch.log2(most / 448)), torch.ones_like(most))
    y = y / scale
    grain = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    n = torch.floor(y.abs() / grain + u.view(-1, BLOCK).double())
    if nonzero:
        n = torch.where(y > 0, n.clamp(min=1), n)
    return (torch.sign(y) * n * grain).view(-1), scale.view(-1)


def _exact_adamw(s):
    case = s["case"]
    s["step"] += 1
    p, g = s["param"].double(), s["grad"].double()
    norm = None
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["clip"] / (float(norm) + 1e-6))
    if case["bits"] == 8:
        m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (s["v"].double() * s["v_scale"].double().repeat_interleave(BLOCK)).square()
    else:
        m, v = s["m"].double(), s["v"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g.square()
    p = p - case["lr"] * 0.01 * p - case["lr"] * (m / (1 - BETA1 ** s["step"])) / (torch.sqrt(v / (1 - BETA2 ** s["step"])) + EPS)
    out = dict(param=p, m=m, v=v, copy=p if case["copy"] else None, norm=norm)
    if case["bits"] == 8:
        um, uv = _rounding(s, p.numel(), p.device)
        out["m"], out["m_scale"] = _exact_8bit(m, um, False)
        out["v"], out["v_scale"] = _exact_8bit(v.sqrt(), uv, True)
    return {k: x for k, x in out.items() if x is not None}


def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "loss": _exact_loss, "adamw": _exact_adamw}[case["op"]](s)
