"""Cases, plain forms and exact values of the embedding, preference-loss and AdamW operators.

`listed()` and `draw()` give cases, `prepare()` makes what a training or serving program has in hand,
`run()` is one pass: the elementary torch form where `own` is false, the framework's calls where it is true.

Sizes are those of the configured tables (7,050 items of 26,495 nodes; 18,357 items; 63,001 items of 255,404
nodes; widths 64 and 128) or generic stacks of dense layers.
"""
import math

import torch

own = False

DEV = "cuda"
IGNORE = -100        # label of a masked position
BLOCK = 64           # elements that share a scale of an 8-bit state
SMALL = 4096         # tensors below this many elements keep 32-bit states
FULL = 448.0         # largest finite value of torch.float8_e4m3fn
TINY = 1e-30         # block maxima below this count as this
STEP0 = 100          # updates that a prepared optimizer state has behind it
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# --------------------------------------------------------------------------------------------- cases
def _emb(name, rows, dim, n, dtype, ids="int64", train=True, pad=False):
    return {"name": name, "op": "embedding", "rows": rows, "dim": dim, "n": n, "dtype": dtype, "ids": ids,
            "train": train, "pad": pad}


def _pref(name, pairs, length, items, dtype):
    return {"name": name, "op": "preference", "pairs": pairs, "length": length, "items": items, "dtype": dtype}


def _adamw(name, rows, dim, layers, hidden, dtype, bits, clip):
    return {"name": name, "op": "adamw", "rows": rows, "dim": dim, "layers": layers, "hidden": hidden,
            "dtype": dtype, "bits": bits, "clip": clip}


def listed():
    return [
        # a serving request: the rows of eight users, no gradient
        _emb("emb_serve", 192403, 64, 8, "float32", train=False),
        # one small training batch of item ids at the smallest catalogue
        _emb("emb_batch", 7050, 64, 512, "float32"),
        # padded interaction histories (64 users, 50 places) over all nodes of the smallest graph
        _emb("emb_histories", 26495, 128, 64 * 50, "bfloat16", pad=True),
        # every training interaction's node of a large batch at the largest graph: long runs of popular ids
        _emb("emb_large", 255404, 128, 1 << 20, "bfloat16", ids="int32"),
        # four pairs of next-item choices over the smallest catalogue
        _pref("pref_next_item", 4, 1, 7050, "float32"),
        # two pairs of short lists over the largest catalogue: few rows, a long axis
        _pref("pref_few_rows", 2, 5, 63001, "float32"),
        # sixteen pairs of lists of up to twenty over a catalogue of odd size
        _pref("pref_lists", 16, 20, 18357, "bfloat16"),
        # a full training batch of lists over the largest catalogue
        _pref("pref_large", 32, 50, 63001, "bfloat16"),
        # the weights of a small network of dense layers, clipped: launch latency
        _adamw("adamw_layers", 0, 0, 8, 64, "float32", 32, 1.0),
        # the id table of the largest graph, states in 8 bits
        _adamw("adamw_table8", 255404, 64, 0, 0, "float32", 8, 0.0),
        # a stack of wide layers in bfloat16 beside a table, states in 8 bits, clipped
        _adamw("adamw_stack8", 63001, 128, 8, 1024, "bfloat16", 8, 1.0),
        # table and wide layers in 32 bits, clipped
        _adamw("adamw_stack32", 255404, 128, 8, 1024, "float32", 32, 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "preference", "adamw"])
    if op == "embedding":
        dim = rng.choice([16, 32, 64, 100, 128, 256, rng.randint(8, 256)])
        n = _log(rng, 8, min(1 << 20, (1 << 27) // dim))
        c = _emb("", _log(rng, 500, 255404), dim, n, rng.choice(list(DTYPES)), rng.choice(["int32", "int64"]),
                 rng.random() < 0.8, rng.random() < 0.5)
    elif op == "preference":
        items = _log(rng, 500, 63001)
        most = max(1, min(3200, 200_000_000 // items))
        length = min(_log(rng, 1, 50), max(1, most // 2))
        c = _pref("", _log(rng, 1, max(1, most // (2 * length))), length, items, rng.choice(["float32", "bfloat16"]))
    else:
        table = rng.random() < 0.6
        layers = rng.randint(1, 8) if not table or rng.random() < 0.5 else 0
        c = _adamw("", _log(rng, 500, 255404) if table else 0, rng.choice([64, 128, rng.randint(8, 128)]) if table else 0,
                   layers, rng.choice([64, 128, 256, rng.randint(33, 1024)]) if layers else 0,
                   rng.choice(["float32", "bfloat16"]), rng.choice([8, 32]), rng.choice([0.0, 1.0]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------- prepare
def _lengths(c):
    """Positions in use of every list of a preference case: from the case alone, between 1 and its length."""
    s = torch.arange(2 * c["pairs"])
    return 1 + (s * 7919 + 13) % c["length"]


def _tensors(c):
    """(shape, decays) of an optimizer case's parameters, the ones with 8-bit states first."""
    every = [((c["rows"], c["dim"]), True)] if c["rows"] else []
    h = c["hidden"]
    for _ in range(c["layers"]):
        every += [((h, h), True), ((4 * h, h), True), ((h, 4 * h), True), ((h,), False), ((4 * h,), False)]
    size = lambda t: math.prod(t[0])  # noqa: E731
    return sorted(every, key=lambda t: size(t) < SMALL) if c["bits"] == 8 else every


def _decode(code, scale):
    return (code.float().view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)


def _encode(x):
    """Values and scales of blocks of 64: the block's largest magnitude becomes the largest float8 value."""
    x = x.view(-1, BLOCK)
    most = x.abs().amax(1, keepdim=True).clamp_min(TINY)
    return (x * (FULL / most)).to(torch.float8_e4m3fn).view(-1), (most / FULL).view(-1)


def _raise_zero(code, x):
    """A root of a second moment that is not zero never becomes zero: at least the smallest float8 value."""
    raw = code.view(torch.uint8)
    return torch.where((x > 0) & (raw == 0), torch.ones_like(raw), raw).view(torch.float8_e4m3fn)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    if case["op"] == "embedding":
        rows, dim, n, dt = case["rows"], case["dim"], case["n"], DTYPES[case["dtype"]]
        # popularity falls with the power -2/3 of the rank, and ranks are spread over the ids
        rank = (rows * torch.rand(n, generator=g, device=DEV).double() ** 3).long().clamp_max(rows - 1)
        ids = torch.randperm(rows, generator=g, device=DEV)[rank]
        if case["pad"]:
            ids = torch.where(torch.rand(n, generator=g, device=DEV) < 0.4, torch.zeros_like(ids), ids)
        s = {"op": "embedding", "weight": (0.1 * normal(rows, dim)).to(dt), "ids": ids.to(getattr(torch, case["ids"])),
             "scale": math.sqrt(dim), "pad": 0 if case["pad"] else None, "train": case["train"]}
        if case["train"]:
            s["weight"].requires_grad_(True)
            s["grad"] = normal(n, dim).to(dt)
        return s
    if case["op"] == "preference":
        lists, length, items, dt = 2 * case["pairs"], case["length"], case["items"], DTYPES[case["dtype"]]
        scores = (2.0 * normal(lists, length, items)).to(dt)
        chosen = torch.randint(items, (lists, length), generator=g, device=DEV)
        used = torch.arange(length, device=DEV) < _lengths(case).to(DEV).unsqueeze(1)
        # what a frozen copy of the model would say: near the lists' own log-probabilities
        ref = used.sum(1) * (-math.log(items) - 2.0) + 2.0 * normal(lists)
        return {"op": "preference", "scores": scores.requires_grad_(True), "ref": ref, "beta": 0.1, "smoothing": 0.1,
                "items": torch.where(used, chosen, torch.full_like(chosen, IGNORE))}
    dt = DTYPES[case["dtype"]]
    tensors = _tensors(case)
    sizes = [math.prod(t[0]) for t in tensors]
    room = [-(-n // BLOCK) * BLOCK for n in sizes]            # every tensor begins at a multiple of 64
    starts = [sum(room[:k]) for k in range(len(room))]
    total = sum(room)
    place = torch.zeros(total, device=DEV)                    # 0 where no parameter lies
    decay = torch.zeros(total // BLOCK, device=DEV)
    for (shape, decays), n, a, r in zip(tensors, sizes, starts, room):
        place[a:a + n] = 1.0
        decay[a // BLOCK:(a + r) // BLOCK] = 0.01 if decays else 0.0
    split = sum(r for n, r in zip(sizes, room) if case["bits"] == 8 and n >= SMALL)
    spread = torch.exp(normal(total))
    first, root = 0.02 * spread * normal(total) * place, 0.05 * spread * (0.5 + torch.rand(total, generator=g, device=DEV)) * place
    s = {"op": "adamw", "shapes": [list(t[0]) for t in tensors], "decays": [t[1] for t in tensors], "sizes": sizes,
         "starts": starts, "split": split, "bits": case["bits"], "clip": case["clip"], "lr": 1e-3, "betas": (0.9, 0.999),
         "eps": 1e-8, "decay": decay, "step": STEP0, "param": (0.1 * normal(total) * place).to(dt),
         "grad": (0.1 * spread * normal(total) * place).to(dt),
         "exp_avg": first[split:].clone(), "exp_avg_sq": root[split:].square()}
    if split:
        s["exp_avg8"], s["exp_avg8_scale"] = _encode(first[:split])
        code, s["exp_avg_sq8_scale"] = _encode(root[:split])
        s["exp_avg_sq8"] = _raise_zero(code, root[:split])
    return s


# ----------------------------------------------------------------------------------------------- run
def run(state):
    op = state["op"]
    if own:
        return {"embedding": _own_embedding, "preference": _own_preference, "adamw": _own_adamw}[op](state)
    return {"embedding": _plain_embedding, "preference": _plain_preference, "adamw": _plain_adamw}[op](state)


def _own_embedding(s):
    from recommend_amd import ops
    if not s["train"]:
        return ops.embedding_lookup(s["weight"], s["ids"], scale=s["scale"], padding_idx=s["pad"])
    out = ops.embedding_lookup(s["weight"], s["ids"], scale=s["scale"], padding_idx=s["pad"])
    return [out.detach(), torch.autograd.grad(out, s["weight"], s["grad"])[0]]


def _plain_embedding(s):
    weight = s["weight"].detach()
    ids = s["ids"].long()
    out = (weight[ids].float() * s["scale"]).to(weight.dtype)
    if not s["train"]:
        return out
    part = s["grad"].float() * s["scale"]
    if s["pad"] is not None:
        part = part * (ids != s["pad"]).float().unsqueeze(1)
    total = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device).index_add_(0, ids, part)
    return [out, total.to(weight.dtype)]


def _own_preference(s):
    from recommend_amd.loss import preference_loss
    loss, logps = preference_loss(s["scores"], s["items"], s["ref"], beta=s["beta"], label_smoothing=s["smoothing"])
    return [loss.detach(), logps.detach(), torch.autograd.grad(loss, s["scores"])[0]]


def _plain_preference(s):
    scores, beta, eps = s["scores"].detach(), s["beta"], s["smoothing"]
    x = scores.float()
    used = s["items"] != IGNORE
    label = torch.where(used, s["items"], torch.zeros_like(s["items"])).unsqueeze(2)
    top = x.amax(2, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(2, keepdim=True)
    logp = ((x.gather(2, label) - top) - torch.log(total)).squeeze(2)
    logps = torch.where(used, logp, torch.zeros_like(logp)).sum(1)
    pairs = logps.shape[0] // 2
    ratio = logps - s["ref"]
    h = beta * (ratio[:pairs] - ratio[pairs:])
    soft = torch.log1p(torch.exp(-h.abs()))
    loss = ((1 - eps) * (soft + (-h).clamp_min(0)) + eps * (soft + h.clamp_min(0))).mean()
    slope = beta / pairs * (eps / (1 + torch.exp(-h)) - (1 - eps) / (1 + torch.exp(h)))
    weight = torch.cat([slope, -slope]).unsqueeze(1) * used.float()
    grad = e * (-weight.unsqueeze(2) / total)
    grad.scatter_add_(2, label, weight.unsqueeze(2))
    return [loss, logps, grad.to(scores.dtype)]


def _own_adamw(s):
    opt = s.get("optimizer")
    if opt is None:                                # a program makes its optimizer once and keeps it
        opt = s["optimizer"] = _make_optimizer(s)
    opt.step()
    return _adamw_outputs(s)


def _make_optimizer(s):
    from recommend_amd.optim import FusedAdamW
    params = []
    for shape, n, a in zip(s["shapes"], s["sizes"], s["starts"]):
        p = torch.nn.Parameter(s["param"][a:a + n].view(shape))
        p.grad = s["grad"][a:a + n].view(shape)
        params.append(p)
    groups = [{"params": [p for p, d in zip(params, s["decays"]) if d is yes], "weight_decay": 0.01 if yes else 0.0}
              for yes in (True, False)]
    opt = FusedAdamW([g for g in groups if g["params"]], lr=s["lr"], betas=s["betas"], eps=s["eps"],
                     max_grad_norm=s["clip"] or None, state_bits=s["bits"], min_8bit_size=SMALL)
    for p, n, a in zip(params, s["sizes"], s["starts"]):
        b = a - s["split"]
        if b >= 0:
            st = {"exp_avg": s["exp_avg"][b:b + n].view(p.shape), "exp_avg_sq": s["exp_avg_sq"][b:b + n].view(p.shape)}
        else:
            e, k, m = a + -(-n // BLOCK) * BLOCK, a // BLOCK, -(-(a + n) // BLOCK)
            st = {"exp_avg8": s["exp_avg8"][a:e], "exp_avg8_scale": s["exp_avg8_scale"][k:m],
                  "exp_avg_sq8": s["exp_avg_sq8"][a:e], "exp_avg_sq8_scale": s["exp_avg_sq8_scale"][k:m]}
        opt.state[p].update(st, step=torch.tensor(float(s["step"])))
    return opt


_STATES = ("exp_avg", "exp_avg_sq", "exp_avg8", "exp_avg8_scale", "exp_avg_sq8", "exp_avg_sq8_scale")


def _adamw_outputs(s):
    return {k: s[k] for k in ("param",) + _STATES if k in s}


def _plain_adamw(s):
    s["step"] += 1
    (b1, b2), split, t = s["betas"], s["split"], s["step"]
    grad = s["grad"].float()
    if s["clip"]:
        # in 64 bits: the norm is a long sum, and the rounding of every state hangs on it
        norm = grad.double().square().sum().sqrt()
        grad = grad * (s["clip"] / (norm + 1e-6)).clamp_max(1.0).float()
    first, second = [s["exp_avg"]], [s["exp_avg_sq"]]
    if split:
        root = _decode(s["exp_avg_sq8"], s["exp_avg_sq8_scale"])
        first, second = [_decode(s["exp_avg8"], s["exp_avg8_scale"])] + first, [root * root] + second
    first = torch.cat(first) * b1 + grad * (1 - b1)
    second = torch.cat(second) * b2 + (grad * grad) * (1 - b2)
    root = torch.sqrt(second)
    p = s["param"].float()
    p = p - (p.view(-1, BLOCK) * (s["lr"] * s["decay"]).unsqueeze(1)).view(-1)
    p = p - (s["lr"] / (1 - b1 ** t)) * (first / (root / math.sqrt(1 - b2 ** t) + s["eps"]))
    s["param"].copy_(p)
    s["exp_avg"].copy_(first[split:])
    s["exp_avg_sq"].copy_(second[split:])
    if split:
        for key, x in (("exp_avg8", first[:split]), ("exp_avg_sq8", root[:split])):
            code, scale = _encode(x)
            s[key].copy_(_raise_zero(code, x) if key == "exp_avg_sq8" else code)
            s[key + "_scale"].copy_(scale)
    return _adamw_outputs(s)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "embedding":
        size = DTYPES[case["dtype"]].itemsize
        row, n = case["dim"] * size, case["n"]
        ids = n * getattr(torch, case["ids"]).itemsize
        b = min(n, case["rows"]) * row + n * row + ids
        if case["train"]:
            b += n * row + case["rows"] * row
        return {"bytes": b, "flops": n * case["dim"] * (2 if case["train"] else 1)}
    if case["op"] == "preference":
        size = DTYPES[case["dtype"]].itemsize
        rows, used = 2 * case["pairs"] * case["length"], int(_lengths(case).sum())
        # masked positions are not read; their gradient is written
        return {"bytes": (rows + used) * case["items"] * size + rows * 8, "flops": 8 * used * case["items"]}
    size = DTYPES[case["dtype"]].itemsize
    b = f = 0
    for shape, _ in _tensors(case):
        n = math.prod(shape)
        state = 4 + 16 / BLOCK if case["bits"] == 8 and n >= SMALL else 16
        b += n * (3 * size + state)
        f += 16 * n
    return {"bytes": b, "flops": f}


# --------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        weight, ids = s["weight"].detach().double(), s["ids"].long()
        out = weight.index_select(0, ids) * s["scale"]
        if not case["train"]:
            return out
        grad = s["grad"].double() * s["scale"]
        if s["pad"] is not None:
            grad[ids == s["pad"]] = 0
        return [out, torch.zeros_like(weight).index_add_(0, ids, grad)]
    if case["op"] == "preference":
        pairs, beta, eps = case["pairs"], s["beta"], s["smoothing"]
        logps = torch.zeros(2 * pairs, dtype=torch.float64, device=DEV)
        grad = torch.zeros(s["scores"].shape, dtype=torch.float64, device=DEV)
        for k in range(2 * pairs):                # a list at a time: 64 bits of every score are large
            at = torch.nonzero(s["items"][k] != IGNORE).squeeze(1)
            pick = s["items"][k][at].unsqueeze(1)
            x = s["scores"].detach()[k][at].double()
            lse = torch.logsumexp(x, 1, keepdim=True)
            logps[k] = (x.gather(1, pick) - lse).sum()
            d = -torch.exp(x - lse)
            d.scatter_add_(1, pick, torch.ones_like(pick, dtype=torch.float64))
            grad[k, at] = d
        h = beta * ((logps - s["ref"].double())[:pairs] - (logps - s["ref"].double())[pairs:])
        loss = -((1 - eps) * torch.nn.functional.logsigmoid(h) + eps * torch.nn.functional.logsigmoid(-h)).mean()
        slope = beta * (eps * torch.sigmoid(h) - (1 - eps) * torch.sigmoid(-h)) / pairs
        return [loss, logps, grad * torch.cat([slope, -slope]).view(-1, 1, 1)]
    (b1, b2), split, t = s["betas"], s["split"], s["step"] + 1
    out = {}
    g, p = s["grad"].double(), s["param"].double()
    if s["clip"]:
        g = g * min(1.0, s["clip"] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    if split:
        both = [s[k].double().view(-1, BLOCK) * s[k + "_scale"].double().view(-1, 1) for k in ("exp_avg8", "exp_avg_sq8")]
        m, v = torch.cat([both[0].view(-1), m]), torch.cat([both[1].view(-1) ** 2, v])
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - s["lr"] * s["decay"].double().repeat_interleave(BLOCK))
    out["param"] = p - s["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + s["eps"])
    out["exp_avg"], out["exp_avg_sq"] = m[split:], v[split:]
    if split:
        # the codes are roundings next to a border: no 64-bit value says on which side; their scales have one
        out["exp_avg8"] = out["exp_avg_sq8"] = None
        out["exp_avg8_scale"] = m[:split].abs().view(-1, BLOCK).amax(1) / FULL
        out["exp_avg_sq8_scale"] = v[:split].sqrt().view(-1, BLOCK).amax(1) / FULL
    return out
