"""More operators of a training step, as cases that can be measured:

  adamw   adamw_step: AdamW over many tensors at once, moments in 32 or in 8 bits
  rotary  rotary and rotary_backward: the position rotation of queries and keys
  qk      qk_norm_rotary and its gradient: per-head norms of queries and keys with the rotation
  logp    token_log_probs and its gradient: log probabilities of given tokens, entropy, top alternatives

`run` computes each in plain torch operations in 32 bits (angles in 64), or, where `own` is true, through this package.
"""
import math

import torch

own = False

IGNORE = -100
BLOCK = 2048
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.95, 1e-8, 0.1


def listed():
    return [
        # The norm gains of the 80 layers of the 70B configuration and its last norm: many small tensors, where latency counts.
        {"name": "adamw gains 70B", "op": "adamw", "tensors": 161, "n": 8192, "odd": 0, "dtype": "bf16", "grad": "bf16", "bits": 32, "master": False},
        # Its embedding and head (32000 x 8192 each) beside the low-rank step, moments in 8 bits.
        {"name": "adamw embedding 70B int8", "op": "adamw", "tensors": 2, "n": 32000 * 8192, "odd": 0, "dtype": "bf16", "grad": "bf16", "bits": 8, "master": False},
        # Adapters and biases of odd sizes, gradients accumulated in fp32, an fp32 master copy.
        {"name": "adamw ragged master", "op": "adamw", "tensors": 57, "n": 1 << 18, "odd": 1, "dtype": "bf16", "grad": "f32", "bits": 32, "master": True},
        # Queries and keys of the 70B configuration (64 + 8 heads of 128) as the qkv product leaves them.
        {"name": "rotary 70B", "op": "rotary", "n": 8192, "hq": 64, "hk": 8, "head": 128, "part": 128, "layout": "half", "dtype": "bf16",
         "scaling": "none", "factor": 1.0, "first": 0, "back": False},
        # The gradient in a context stretched 32 times, far positions, interleaved pairs, part of the head, an odd length.
        {"name": "rotary back long ragged f16", "op": "rotary", "n": 2047, "hq": 32, "hk": 8, "head": 96, "part": 64, "layout": "interleaved", "dtype": "f16",
         "scaling": "yarn", "factor": 32.0, "first": 128000, "back": True},
        # One token of a generation: the smallest call.
        {"name": "qk one token", "op": "qk", "n": 1, "hq": 64, "hk": 8, "head": 128, "part": 128, "layout": "half", "dtype": "bf16",
         "scaling": "none", "factor": 1.0, "first": 4095, "back": False},
        {"name": "qk 70B", "op": "qk", "n": 8192, "hq": 64, "hk": 8, "head": 128, "part": 128, "layout": "half", "dtype": "bf16",
         "scaling": "none", "factor": 1.0, "first": 0, "back": False},
        # The gradient of a long micro-batch, with the gradients of the two gains.
        {"name": "qk back 70B", "op": "qk", "n": 8192, "hq": 64, "hk": 8, "head": 128, "part": 128, "layout": "half", "dtype": "bf16",
         "scaling": "none", "factor": 1.0, "first": 0, "back": True},
        # Policy-gradient training at the 7B head, an eighth masked: log probabilities, entropy, both gradients.
        {"name": "logp 7B step", "op": "logp", "n": 4096, "d": 4096, "v": 32000, "top": 0, "dtype": "bf16", "masked": 0.125, "mode": "train"},
        # A teacher's answers at the 70B head: eight alternatives for each token.
        {"name": "logp 70B top", "op": "logp", "n": 8192, "d": 8192, "v": 32000, "top": 8, "dtype": "bf16", "masked": 0.0, "mode": "score"},
        # One token of a generation with the twenty alternatives that an interface shows.
        {"name": "logp one token top", "op": "logp", "n": 1, "d": 4096, "v": 32000, "top": 20, "dtype": "bf16", "masked": 0.0, "mode": "score"},
        # Short answers in fp16 over a large, odd vocabulary.
        {"name": "logp ragged f16", "op": "logp", "n": 311, "d": 2048, "v": 131071, "top": 5, "dtype": "f16", "masked": 0.5, "mode": "train"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adamw", "rotary", "qk", "logp", "logp"])
    if op == "adamw":
        tensors = _log_int(rng, 1, 300)
        bits = rng.choice([32, 8])
        return {"op": op, "tensors": tensors, "n": _log_int(rng, 1, 32000 * 8192 // tensors), "odd": rng.choice([0, 1]), "dtype": rng.choice(["bf16", "f16", "f32"]),
                "grad": rng.choice(["bf16", "f32"]), "bits": bits, "master": False}
    n = _log_int(rng, 1, 8192)
    if op in ("rotary", "qk"):
        hk = rng.choice([1, 4, 8])
        head = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
        return {"op": op, "n": n, "hq": hk * rng.randint(1, 8), "hk": hk, "head": head, "part": rng.choice([head, head // 2]), "layout": rng.choice(["half", "interleaved"]),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "factor": float(rng.choice([2, 8, 32])),
                "first": _log_int(rng, 1, 1 << 20), "back": rng.random() < 0.5}
    d, v = 8 * _log_int(rng, 8, 1024), _log_int(rng, 257, 131071)
    while n * v > 8192 * 32000 or n * v * d > 4096 * 32000 * 4096:
        v = v * 3 // 4
    masked = rng.choice([0.0, 0.0, rng.uniform(0.05, 0.9)])
    return {"op": op, "n": n, "d": d, "v": v, "top": rng.choice([0, 1, 5, 20, 32]), "dtype": rng.choice(["bf16", "bf16", "f16"]), "masked": round(masked, 3),
            "mode": rng.choice(["train", "hidden", "score", "score"])}


# ---- inputs ----
def _sizes(case):
    """Elements of each tensor: all n, or odd ones between n / 16 and n."""
    if not case["odd"]:
        return [case["n"]] * case["tensors"]
    return [max(1, case["n"] // (1 + i % 16) - 37 * i) for i in range(case["tensors"])]


def _blocks(case):
    return [-(-n // BLOCK) for n in _sizes(case)]


def _maps():
    """The signed and the unsigned dynamic map of 8-bit moments (256 sorted values each): a sign, 0 to 6 zeros that give
    the decade, and a fraction of the bits that are left, at the middle of equal parts of 0.1 to 1; and 0 and 1."""
    out = []
    for signed in (True, False):
        bits, got = 7 if signed else 8, [0.0, 1.0]
        for i in range(7):
            parts = 2 ** (i + bits - 7)
            for j in range(parts):
                x = 10.0 ** (i - 6) * (0.1 + 0.9 * (j + 0.5) / parts)
                got += [x, -x] if signed else [x]
        out.append(sorted(got))
    return out


def _inv_freq(case):
    """Angle for each position and pair, in 64 bits."""
    r, base, s = case["part"], 10000.0, case["factor"]
    if case["scaling"] == "ntk":
        base *= s ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "yarn":  # turns in the 4096 positions of training: kept above 32, divided below 1
        keep = ((4096 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * keep + f / s * (1 - keep)
    return f


def _attention(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "yarn" else 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "adamw":
        sizes, total = _sizes(case), BLOCK * sum(_blocks(case))
        starts = [0]
        for b in _blocks(case):
            starts.append(starts[-1] + b * BLOCK)
        inside = torch.zeros(total, dtype=torch.bool, device="cuda")
        for a, n in zip(starts, sizes):
            inside[a:a + n] = True
        flat = (0.02 * normal(total)).masked_fill_(~inside, 0.0)
        grad = (1e-3 * normal(total)).masked_fill_(~inside, 0.0)
        m, v = (3e-4 * normal(total)).masked_fill_(~inside, 0.0), (1e-6 * normal(total).square()).masked_fill_(~inside, 0.0)
        s["flat"], grads = flat.to(TYPES[case["dtype"]]), grad.to(TYPES[case["grad"]])
        s["params"] = [s["flat"][a:a + n] for a, n in zip(starts, sizes)]
        s["grads"] = [grads[a:a + n] for a, n in zip(starts, sizes)]
        s["master"] = s["flat"].float() if case["master"] else None
        s["clip"] = torch.tensor(0.7, device="cuda")
        s["step"] = torch.tensor(100, dtype=torch.int64, device="cuda")
        if case["bits"] == 32:
            s["m"], s["v"], s["ms"], s["vs"] = m, v, None, None
        else:
            s["maps"] = [torch.tensor(x, dtype=torch.float64, device="cuda").float() for x in _maps()]
            s["m"], s["ms"] = _encode(m, s["maps"][0])
            s["v"], s["vs"] = _encode(v, s["maps"][1])
        return s
    dt, n = TYPES[case["dtype"]], case["n"]
    if case["op"] in ("rotary", "qk"):
        hq, hk, d = case["hq"], case["hk"], case["head"]
        # as the qkv product leaves them: queries, keys and values of a token side by side
        qkv = normal(n, hq + 2 * hk, d).to(dt)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        s["positions"] = case["first"] + torch.arange(n, device="cuda")
        s["inv_freq"] = _inv_freq(case)
        if case["op"] == "qk":
            s["wq"], s["wk"] = ((1.0 + 0.1 * normal(d)).to(dt) for _ in range(2))
        if case["back"]:
            s["dq"], s["dk"] = (1e-3 * normal(n, hq, d)).to(dt), (1e-3 * normal(n, hk, d)).to(dt)
        return s
    # Weights and states on a grid, so that sums of their products are exact in 32 bits in any order: which of two
    # alternatives is the better one then has one answer, ties included.
    d, v = case["d"], case["v"]
    w = (16 * normal(v, d)).round_().clamp_(-64, 64) * 2.0 ** -10
    labels = torch.randint(0, v, (n,), generator=gen, device="cuda")
    known = w[labels]
    lift = 10.0 * torch.rand(n, 1, generator=gen, device="cuda")  # a head that knows some of its labels
    h = ((normal(n, d) + lift * known / known.square().sum(1, keepdim=True)) * 8).round_().clamp_(-32, 32) / 8
    out = torch.rand(n, generator=gen, device="cuda") < case["masked"]
    out[0] = False
    labels[out] = IGNORE
    h[out & (torch.arange(n, device="cuda") % 3 == 0)] = float("nan")  # nothing is said about masked rows
    s.update(hidden=h.to(dt), weight=w.to(dt), labels=labels)
    if case["mode"] != "score":  # advantages, and a bonus for entropy
        s["grad"] = -normal(n) / n
        s["grad_entropy"] = torch.full((n,), -0.01 / n, device="cuda")
    return s


# ---- plain forms ----
def _encode(x, codes):
    """Blocks of x against their largest magnitude: the place of the nearest value (the lower of two as near), scales.
    A block below the smallest normal number is all zeros."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1)
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    x = x * torch.where(scale > 0, 1.0 / scale, scale)[:, None]
    at = torch.searchsorted(codes, x).clamp_(1, 255)
    at = at - 1 + ((codes[at] - x).abs() < (x - codes[at - 1]).abs()).long()
    return at.to(torch.uint8).view(torch.int8).view(-1), scale


def _decode(q, scale, codes):
    return (codes[q.view(torch.uint8).view(-1, BLOCK).int()] * scale[:, None]).view(-1)


def _padded(tensors):
    """The tensors one after the other in 32 bits, each filled up to whole blocks."""
    return torch.cat([torch.nn.functional.pad(t.float(), (0, -t.numel() % BLOCK)) for t in tensors])


def _plain_adamw(s):
    eight = s["case"]["bits"] == 8
    m = _decode(s["m"], s["ms"], s["maps"][0]) if eight else s["m"]
    v = _decode(s["v"], s["vs"], s["maps"][1]) if eight else s["v"]
    p = s["master"] if s["case"]["master"] else s["flat"].float()
    s["step"] += 1
    t = s["step"].double()
    first, second = 1.0 / (1.0 - BETA1 ** t), 1.0 / (1.0 - BETA2 ** t)
    g = _padded(s["grads"]) * s["clip"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = p - LR * (m * first.float() / (torch.sqrt(v * second.float()) + ADAM_EPS) + DECAY * p)
    s["flat"].copy_(p)
    out = {"params": s["flat"]}
    if s["case"]["master"]:
        s["master"].copy_(p)
        out["master"] = s["master"]
    if eight:
        (q, scale), (r, vscale) = _encode(m, s["maps"][0]), _encode(v, s["maps"][1])
        s["m"].copy_(q), s["v"].copy_(r), s["ms"].copy_(scale), s["vs"].copy_(vscale)
        out["m"], out["v"] = _decode(q, scale, s["maps"][0]), _decode(r, vscale, s["maps"][1])
    else:
        out["m"], out["v"] = s["m"].copy_(m), s["v"].copy_(v)
    return out


def _rotate(x, s, back=False):
    """x (tokens, heads, head) in 32 bits, rotated (or turned back)."""
    r = s["case"]["part"]
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]
    a = _attention(s["case"])
    cos, sin = (torch.cos(angle) * a).float(), (torch.sin(angle) * (-a if back else a)).float()
    if s["case"]["layout"] == "half":
        u, v = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([u * cos - v * sin, v * cos + u * sin, x[..., r:]], 2)
    u, v = x[..., :r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([u * cos - v * sin, v * cos + u * sin], 3).flatten(2), x[..., r:]], 2)


def _plain_rotary(s):
    back = s["case"]["back"]
    dt = s["q"].dtype
    q, k = (s["dq"], s["dk"]) if back else (s["q"], s["k"])
    return {"q": _rotate(q.float(), s, back).to(dt), "k": _rotate(k.float(), s, back).to(dt)}


def _norm_back(dy, x, w, s):
    x, w, g = x.float(), w.float(), _rotate(dy.float(), s, True)
    r = torch.rsqrt(x.square().mean(2, keepdim=True) + EPS)
    dx = r * (w * g) - x * (r * r * r * (w * g * x).mean(2, keepdim=True))
    return dx.to(dy.dtype), (g * x * r).sum((0, 1))


def _plain_qk(s):
    if s["case"]["back"]:
        (dq, dwq), (dk, dwk) = _norm_back(s["dq"], s["q"], s["wq"], s), _norm_back(s["dk"], s["k"], s["wk"], s)
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    q, k = s["q"].float(), s["k"].float()
    q = q * torch.rsqrt(q.square().mean(2, keepdim=True) + EPS) * s["wq"].float()
    k = k * torch.rsqrt(k.square().mean(2, keepdim=True) + EPS) * s["wk"].float()
    return {"q": _rotate(q, s).to(s["q"].dtype), "k": _rotate(k, s).to(s["k"].dtype)}


def _plain_logp(s):
    case = s["case"]
    keep = s["labels"] != IGNORE
    at = torch.where(keep, s["labels"], torch.zeros_like(s["labels"]))[:, None]
    h = s["hidden"].float().masked_fill(~keep[:, None], 0.0)
    w = s["weight"].float()
    logits = h @ w.T
    top = logits.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    out = {}
    if case["top"]:
        best, ids = torch.sort(logits, dim=1, descending=True, stable=True)
        out["top_log_probs"] = (best[:, :case["top"]] - lse).masked_fill(~keep[:, None], 0.0)
        out["top_ids"] = ids[:, :case["top"]].masked_fill(~keep[:, None], -1)
        del best, ids
    logits = logits.sub_(lse)  # log probabilities
    p = torch.exp(logits)
    entropy = -(p * logits).sum(1)
    out["log_probs"] = logits.gather(1, at)[:, 0].masked_fill(~keep, 0.0)
    out["entropy"] = entropy.masked_fill(~keep, 0.0)
    if case["mode"] == "score":
        return out
    a, b = (s[x].masked_fill(~keep, 0.0)[:, None] for x in ("grad", "grad_entropy"))
    g = -p * (a + b * (logits + entropy[:, None]))
    g.scatter_add_(1, at, a)
    out["d_hidden"] = (g @ w).to(s["hidden"].dtype)
    if case["mode"] == "train":
        out["d_weight"] = (g.T @ h).to(s["weight"].dtype)
    return out


# ---- the framework's ----
def _own_adamw(s):
    import aethelstream_b200 as A
    state = A.AdamWState(s["m"], s["v"], s["ms"], s["vs"], s["master"], s["step"])
    config = A.AdamWConfig(beta1=BETA1, beta2=BETA2, eps=ADAM_EPS, lr=LR, weight_decay=DECAY)
    A.adamw_step(s["params"], s["grads"], state, config, clip=s["clip"])
    out = {"params": s["flat"]}
    if s["master"] is not None:
        out["master"] = s["master"]
    out["m"], out["v"] = A.adamw_moments(state)
    return out


def _plan(s):
    """The rotation's plan, which a program makes once."""
    if "plan" not in s:
        import aethelstream_b200 as A
        case = s["case"]
        s["plan"] = A.RotaryPlan(case["part"], base=10000.0, layout=case["layout"], scaling=case["scaling"], factor=case["factor"], original_length=4096, device="cuda")
    return s["plan"]


def _own_rotary(s):
    import aethelstream_b200 as A
    if s["case"]["back"]:
        q, k = A.rotary_backward(s["dq"], s["dk"], s["positions"], _plan(s))
    else:
        q, k = A.rotary(s["q"], s["k"], s["positions"], _plan(s))
    return {"q": q, "k": k}


def _own_qk(s):
    import aethelstream_b200 as A
    if s["case"]["back"]:
        dq, dk, dwq, dwk = A.qk_norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], s["wq"], s["wk"], s["positions"], _plan(s), eps=EPS)
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    q, k = A.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["positions"], _plan(s), eps=EPS)
    return {"q": q, "k": k}


def _own_logp(s):
    import aethelstream_b200 as A
    mode, top = s["case"]["mode"], s["case"]["top"]
    r = A.token_log_probs(s["hidden"], s["weight"], s["labels"], top_k=top, ignore_index=IGNORE)
    out = {"log_probs": r.log_probs, "entropy": r.entropy}
    if top:
        out["top_log_probs"], out["top_ids"] = r.top_log_probs, r.top_ids
    if mode != "score":
        dh, dw = A.token_log_probs_backward(s["hidden"], s["weight"], s["labels"], r, grad_log_probs=s["grad"], grad_entropy=s["grad_entropy"], ignore_index=IGNORE,
                                            need_weight=mode == "train")
        out["d_hidden"] = dh
        if mode == "train":
            out["d_weight"] = dw
    return out


PLAIN = {"adamw": _plain_adamw, "rotary": _plain_rotary, "qk": _plain_qk, "logp": _plain_logp}
OWN = {"adamw": _own_adamw, "rotary": _own_rotary, "qk": _own_qk, "logp": _own_logp}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


def work(case):
    if case["op"] == "adamw":
        n, b = sum(_sizes(case)), sum(_blocks(case))
        moved = n * (2 * SIZE[case["dtype"]] + SIZE[case["grad"]])
        moved += n * (8 - SIZE[case["dtype"]]) if case["master"] else 0  # the master copy is read in the parameters' place
        # moments read and written; in 8 bits their scales too, and the values that they stand for are given out
        moved += n * 16 if case["bits"] == 32 else n * 4 + 16 * b + 8 * n
        return {"bytes": moved, "flops": 16.0 * n}
    b = SIZE[case["dtype"]]
    if case["op"] in ("rotary", "qk"):
        rows = case["n"] * (case["hq"] + case["hk"])
        three = case["op"] == "qk" and case["back"]  # the gradient reads x beside dy
        return {"bytes": rows * case["head"] * b * (3 if three else 2) + 8 * case["n"], "flops": rows * case["head"] * (14.0 if three else 7.0 if case["op"] == "qk" else 3.0)}
    n, d, v, mode = case["n"], case["d"], case["v"], case["mode"]
    live = n * (1.0 - case["masked"])  # masked rows' hidden states need not be read
    moved = b * (live * d + v * d) + 16 * n + 12 * n * case["top"]
    moved += b * n * d + 8 * n if mode != "score" else 0
    moved += b * v * d if mode == "train" else 0
    return {"bytes": moved, "flops": 2.0 * {"score": 1, "hidden": 2, "train": 3}[mode] * live * v * d + 6.0 * live * v}


# ---- the definitions in 64 bits, gradients by differentiation ----
def _exact_adamw(case, s):
    t = int(s["step"]) + 1
    sizes, blocks = _sizes(case), _blocks(case)
    ends = torch.tensor(blocks, device="cuda").cumsum(0) * BLOCK
    first = ends - torch.tensor(blocks, device="cuda") * BLOCK
    g = torch.zeros(int(ends[-1]), dtype=torch.float64, device="cuda")
    for a, n, x in zip(first.tolist(), sizes, s["grads"]):
        g[a:a + n] = x.double()
    g *= s["clip"].double()

    def moment(name, which):
        if case["bits"] == 32:
            return s[name].double()
        places = torch.arange(g.numel(), device="cuda") // BLOCK
        return s["maps"][which].double()[s[name].long() % 256] * s[name + "s"].double()[places]

    m = BETA1 * moment("m", 0) + (1 - BETA1) * g
    v = BETA2 * moment("v", 1) + (1 - BETA2) * g ** 2
    p = (s["master"] if case["master"] else s["flat"]).double()
    p = (1 - LR * DECAY) * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + ADAM_EPS)
    out = {"params": p}
    if case["master"]:
        out["master"] = p
    # 8 bits hold the map's value nearest to the moment in 32 bits: next to a border that has no 64-bit counterpart
    out["m"], out["v"] = (None, None) if case["bits"] == 8 else (m, v)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    if case["op"] == "logp":
        rows = torch.nonzero(s["labels"] != IGNORE)[:, 0]
        h = s["hidden"][rows].double().requires_grad_(True)
        w = s["weight"].double().requires_grad_(True)
        n, mode = case["n"], case["mode"]
        logits = h @ w.T
        logs = torch.log_softmax(logits, 1)
        lp, ent = logs[torch.arange(rows.numel(), device="cuda"), s["labels"][rows]], -(logs.exp() * logs).sum(1)

        def whole(x, fill=0.0):
            y = torch.full((n, *x.shape[1:]), fill, dtype=x.dtype, device="cuda")
            y[rows] = x.detach()
            return y

        out = {"log_probs": whole(lp), "entropy": whole(ent)}
        if case["top"]:
            ids = torch.argsort(logits.detach(), dim=1, descending=True, stable=True)[:, :case["top"]]
            out["top_log_probs"], out["top_ids"] = whole(logs.detach().gather(1, ids)), whole(ids, -1)
        if mode != "score":
            (lp * s["grad"][rows].double() + ent * s["grad_entropy"][rows].double()).sum().backward()
            out["d_hidden"] = whole(h.grad)
            if mode == "train":
                out["d_weight"] = w.grad
        return out
    # the rotation as a product of complex numbers
    r = case["part"]
    turn = _attention(case) * torch.exp(1j * (s["positions"].double()[:, None] * s["inv_freq"]))[:, None, :]

    def rotate(x):
        head, rest = x[..., :r], x[..., r:]
        pairs = head.reshape(*x.shape[:2], 2, r // 2).transpose(2, 3) if case["layout"] == "half" else head.reshape(*x.shape[:2], r // 2, 2)
        y = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
        y = y.transpose(2, 3) if case["layout"] == "half" else y
        return torch.cat([y.reshape(*x.shape[:2], r), rest], 2)

    def through(x, w, dy):
        x = x.double().requires_grad_(True)
        w = None if w is None else w.double().requires_grad_(True)
        y = rotate(x if w is None else x / torch.sqrt((x * x).sum(2, keepdim=True) / case["head"] + EPS) * w)
        if dy is None:
            return y.detach(), None
        (y * dy.double()).sum().backward()
        return x.grad, None if w is None else w.grad

    (q, wq), (k, wk) = through(s["q"], s.get("wq"), s.get("dq")), through(s["k"], s.get("wk"), s.get("dk"))
    if case["op"] == "qk" and case["back"]:
        return {"dq": q, "dk": k, "dwq": wq, "dwk": wk}
    return {"q": q, "k": k}
