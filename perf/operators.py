"""The training operators around the optimizer step, as cases that can be measured:

  head     cut_cross_entropy and its gradient: the loss at the language model's head
  store    rms_norm_checkpoint and checkpoint_decode: the first pass's norm, its input kept in 8 bits, and its restoring
  back     rms_norm_checkpoint_backward: the norm's gradient from the 8-bit checkpoint
  wgrad    checkpoint_weight_grad: a linear layer's weight gradient from the 8-bit checkpoint

`run` computes each in plain torch operations in 32 bits, or, where `own` is true, through this package.
"""
import math

import torch

own = False

IGNORE = -100
BLOCK = 128
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # One micro-batch of the 7B configuration (d = 4096) at its 32000-entry head, an eighth of the tokens masked
        # (prompts, padding): loss, gradient of the hidden states and of the head's weight.
        {"name": "head 7B step", "op": "head", "n": 4096, "d": 4096, "v": 32000, "dtype": "bf16", "masked": 0.125, "mode": "train"},
        # The 70B configuration's head (d = 8192) at a long micro-batch: the largest call of a training step.
        {"name": "head 70B step", "op": "head", "n": 8192, "d": 8192, "v": 32000, "dtype": "bf16", "masked": 0.0, "mode": "train"},
        # A frozen head over a large, odd vocabulary at the 13B configuration's width (d = 5120): the hidden states'
        # gradient alone.
        {"name": "head frozen 131071", "op": "head", "n": 2047, "d": 5120, "v": 131071, "dtype": "bf16", "masked": 0.0, "mode": "hidden"},
        # One token scored, as an evaluation that steps through a text does: latency and one read of the weight.
        {"name": "head one token", "op": "head", "n": 1, "d": 4096, "v": 32000, "dtype": "bf16", "masked": 0.0, "mode": "score"},
        # Fine-tuning on short answers in fp16: an odd batch of which most is masked, with garbage (NaN) in the
        # masked rows' hidden states.
        {"name": "head ragged f16", "op": "head", "n": 777, "d": 2048, "v": 50001, "dtype": "f16", "masked": 0.6, "mode": "train"},
        # The first pass at the 70B width: residual add, norm, the sum kept in 8 bits; then its restoring.
        {"name": "store 70B", "op": "store", "n": 8192, "d": 8192, "dtype": "bf16", "residual": True},
        # One token through one norm: the smallest call.
        {"name": "store one token", "op": "store", "n": 1, "d": 4096, "dtype": "bf16", "residual": False},
        # fp32 activations of a reference-mode run, odd length, a last block of the features that is not whole.
        {"name": "store ragged f32", "op": "store", "n": 2047, "d": 1000, "dtype": "f32", "residual": False},
        # The second pass's norm backward at the 70B width, joined with the residual stream's gradient.
        {"name": "back 70B", "op": "back", "n": 8192, "d": 8192, "dtype": "bf16", "residual": True},
        # A short fp16 sequence of odd length at the 13B width.
        {"name": "back ragged f16", "op": "back", "n": 333, "d": 5120, "dtype": "f16", "residual": False},
        # The gate projection of the 7B configuration: dW from the MLP norm's checkpoint.
        {"name": "wgrad 7B gate", "op": "wgrad", "n": 4096, "m": 11008, "d": 4096, "dtype": "bf16", "norm": True},
        # The k/v projection of the 70B configuration, an odd and short batch in fp16, from a plain checkpoint.
        {"name": "wgrad 70B kv ragged", "op": "wgrad", "n": 1001, "m": 1024, "d": 8192, "dtype": "f16", "norm": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["head", "head", "store", "back", "wgrad"])
    n = _log_int(rng, 1, 8192)
    if op == "head":
        # any hidden width that 16 bits make a multiple of 16 bytes, any vocabulary
        d, v = 8 * _log_int(rng, 8, 1024), _log_int(rng, 257, 131071)
        while n * v > 8192 * 32000 or n * v * d > 8192 * 32000 * 8192:
            v = v * 3 // 4
        masked = rng.choice([0.0, 0.0, rng.uniform(0.05, 0.9), 1.0 if n < 64 else 0.0])
        return {"op": op, "n": n, "d": d, "v": v, "dtype": rng.choice(["bf16", "bf16", "f16"]), "masked": round(masked, 3),
                "mode": rng.choice(["train", "train", "hidden", "score"])}
    if op in ("store", "back"):
        return {"op": op, "n": n, "d": _log_int(rng, 33, 8192), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "residual": rng.random() < 0.5}
    return {"op": op, "n": n, "m": 8 * _log_int(rng, 8, 1376), "d": 8 * _log_int(rng, 8, 1024),
            "dtype": rng.choice(["bf16", "bf16", "f16"]), "norm": rng.random() < 0.5}


# ---- inputs ----
def _residual_stream(gen, n, d, dtype):
    """Activations as a block's residual stream has them: unit normal, a few channels tens of times larger."""
    x = torch.randn(n, d, generator=gen, device="cuda")
    gain = torch.ones(d, device="cuda")
    hot = torch.randint(0, d, (max(1, d // 256),), generator=gen, device="cuda")
    gain[hot] = 25.0
    return (x * gain).to(dtype)


def _quantize(x):
    """Codes (int8) and scales (f32) of blocks of BLOCK features, as the checkpoint holds them."""
    n, d = x.shape
    blocks = -(-d // BLOCK)
    p = torch.zeros(n, blocks * BLOCK, device=x.device)
    p[:, :d] = x.float()
    p = p.view(n, blocks, BLOCK)
    amax = p.abs().amax(2)
    scale = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
    v = p * (1.0 / scale)[:, :, None]
    q = torch.trunc(v)
    q = q + torch.sign(v) * ((v - q).abs() >= 0.5)
    return q.clamp(-127, 127).to(torch.int8).view(n, -1)[:, :d].contiguous(), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, n, d = TYPES[case["dtype"]], case["n"], case["d"]
    s = {"case": case, "dtype": dt}
    if case["op"] == "head":
        v = case["v"]
        w = torch.randn(v, d, generator=gen, device="cuda") * 0.02
        labels = torch.randint(0, v, (n,), generator=gen, device="cuda")
        # a head that knows some of its labels: their logits are raised by 0 to 10
        known = w[labels]
        lift = 10.0 * torch.rand(n, 1, generator=gen, device="cuda")
        h = torch.randn(n, d, generator=gen, device="cuda") + lift * known / known.square().sum(1, keepdim=True)
        out = torch.rand(n, generator=gen, device="cuda") < case["masked"]
        labels[out] = IGNORE
        h[out & (torch.arange(n, device="cuda") % 3 == 0)] = float("nan")  # nothing is said about masked rows
        s.update(hidden=h.to(dt), weight=w.to(dt), labels=labels)
        return s
    x = _residual_stream(gen, n, d, dt)
    s["gain"] = (1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dt)
    if case["op"] == "store":
        s["x"] = x
        s["residual"] = _residual_stream(gen, n, d, dt) if case["residual"] else None
        return s
    s["codes"], s["scales"] = _quantize(x)
    rows = case["m"] if case["op"] == "wgrad" else d
    s["dy"] = (1e-3 * torch.randn(n, rows, generator=gen, device="cuda") * torch.exp(torch.randn(n, 1, generator=gen, device="cuda"))).to(dt)
    if case["op"] == "back":
        s["d_residual"] = (1e-3 * torch.randn(n, d, generator=gen, device="cuda")).to(dt) if case["residual"] else None
    return s


# ---- plain forms ----
def _plain_head(s):
    mode, dt = s["case"]["mode"], s["dtype"]
    keep = s["labels"] != IGNORE
    at = torch.where(keep, s["labels"], torch.zeros_like(s["labels"]))[:, None]
    h = s["hidden"].float().masked_fill(~keep[:, None], 0.0)
    w = s["weight"].float()
    logits = h @ w.T
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    losses = (lse - logits.gather(1, at))[:, 0].masked_fill(~keep, 0.0)
    count = keep.sum().clamp(min=1).float()
    out = {"loss": losses.sum() / count, "losses": losses}
    if mode == "score":
        return out
    g = e.div_(total)
    g.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    g.mul_((keep.float() / count)[:, None])
    out["d_hidden"] = (g @ w).to(dt)
    if mode == "train":
        out["d_weight"] = (g.T @ h).to(dt)
    return out


def _restore(s):
    d = s["case"]["d"]
    return s["codes"].float() * s["scales"].repeat_interleave(BLOCK, 1)[:, :d]


def _plain_store(s):
    dt = s["dtype"]
    x = s["x"].float()
    out = {}
    if s["residual"] is not None:
        out["sum"] = (x + s["residual"].float()).to(dt)
        x = out["sum"].float()
    r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    out["y"] = (x * r * s["gain"].float()).to(dt)
    codes, out["scales"] = _quantize(x)
    out["restored"] = (codes.float() * out["scales"].repeat_interleave(BLOCK, 1)[:, :x.shape[1]]).to(dt)
    return out


def _plain_back(s):
    dt = s["dtype"]
    x, dy, w = _restore(s), s["dy"].float(), s["gain"].float()
    r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    dyw = dy * w
    dx = r * dyw - x * (r * r * r * (dyw * x).mean(1, keepdim=True))
    if s["d_residual"] is not None:
        dx = dx + s["d_residual"].float()
    return {"dx": dx.to(dt), "d_weight": (dy * x * r).sum(0)}


def _plain_wgrad(s):
    x = _restore(s)
    if s["case"]["norm"]:
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * s["gain"].float()
    return {"d_weight": (s["dy"].float().T @ x).to(s["dtype"])}


# ---- the framework's ----
def _own_head(s):
    import aethelstream_b200 as A
    mode = s["case"]["mode"]
    ce = A.cut_cross_entropy(s["hidden"], s["weight"], s["labels"], ignore_index=IGNORE)
    out = {"loss": ce.loss, "losses": ce.losses}
    if mode != "score":
        dh, dw = A.cut_cross_entropy_backward(s["hidden"], s["weight"], s["labels"], ce, ignore_index=IGNORE, need_weight=mode == "train")
        out["d_hidden"] = dh
        if mode == "train":
            out["d_weight"] = dw
    return out


def _own_store(s):
    import aethelstream_b200 as A
    out = {}
    if s["residual"] is not None:
        out["y"], ckpt, out["sum"] = A.rms_norm_checkpoint(s["x"], s["gain"], eps=EPS, residual=s["residual"])
    else:
        out["y"], ckpt = A.rms_norm_checkpoint(s["x"], s["gain"], eps=EPS)
    out["scales"] = ckpt.scales
    out["restored"] = A.checkpoint_decode(ckpt)
    return out


def _own_back(s):
    import aethelstream_b200 as A
    ckpt = A.ActivationCheckpoint(s["codes"], s["scales"], s["dtype"])
    dx, dw = A.rms_norm_checkpoint_backward(s["dy"], ckpt, s["gain"], eps=EPS, d_residual=s["d_residual"])
    return {"dx": dx, "d_weight": dw}


def _own_wgrad(s):
    import aethelstream_b200 as A
    ckpt = A.ActivationCheckpoint(s["codes"], s["scales"], s["dtype"])
    return {"d_weight": A.checkpoint_weight_grad(s["dy"], ckpt, norm_weight=s["gain"] if s["case"]["norm"] else None, eps=EPS)}


PLAIN = {"head": _plain_head, "store": _plain_store, "back": _plain_back, "wgrad": _plain_wgrad}
OWN = {"head": _own_head, "store": _own_store, "back": _own_back, "wgrad": _own_wgrad}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


def work(case):
    n, d, b = case["n"], case["d"], SIZE[case["dtype"]]
    scales = 4 * n * -(-d // BLOCK)
    if case["op"] == "head":
        v, mode = case["v"], case["mode"]
        live = n * (1.0 - case["masked"])  # masked rows' hidden states need not be read
        products = {"score": 1, "hidden": 2, "train": 3}[mode]
        moved = b * (live * d + v * d) + 8 * n + 4 * n
        moved += b * n * d if mode != "score" else 0
        moved += b * v * d if mode == "train" else 0
        return {"bytes": moved, "flops": 2.0 * products * live * v * d + 4.0 * live * v}
    if case["op"] == "store":
        sums = 2 if case["residual"] else 0  # the residual read, the sum written
        # read x, write y, codes and scales; the restoring reads codes and scales and writes the values
        return {"bytes": n * d * (b * (3 + sums) + 2) + 2 * scales + b * d, "flops": 12.0 * n * d}
    if case["op"] == "back":
        return {"bytes": n * d * (1 + b * (3 if case["residual"] else 2)) + scales + b * d + 4 * d, "flops": 14.0 * n * d}
    m = case["m"]
    return {"bytes": n * d + scales + b * n * m + b * m * d, "flops": 2.0 * n * m * d}


# ---- the definitions in 64 bits, gradients by differentiation ----
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "head":
        rows = torch.nonzero(s["labels"] != IGNORE)[:, 0]
        h = s["hidden"][rows].double().requires_grad_(True)
        w = s["weight"].double().requires_grad_(True)
        n, mode = case["n"], case["mode"]
        losses = torch.zeros(n, dtype=torch.float64, device="cuda")
        per = -torch.log_softmax(h @ w.T, 1)[torch.arange(rows.numel(), device="cuda"), s["labels"][rows]]
        mean = per.sum() / max(1, rows.numel())
        losses[rows] = per.detach()
        out = {"loss": mean.detach(), "losses": losses}
        if mode != "score":
            mean.backward()
            dh = torch.zeros(n, case["d"], dtype=torch.float64, device="cuda")
            dh[rows] = h.grad
            out["d_hidden"] = dh
            if mode == "train":
                out["d_weight"] = w.grad
        return out
    n, d = case["n"], case["d"]
    gain = s["gain"].double()

    def norm(x):
        return x / torch.sqrt((x * x).sum(1, keepdim=True) / d + EPS)

    if case["op"] == "store":
        x, out = s["x"].double(), {}
        if s["residual"] is not None:
            out["sum"] = x + s["residual"].double()
            x = out["sum"].to(s["dtype"]).double()  # the stored sum is what is normalised and kept
        out["y"] = norm(x) * gain
        edges = [(a, min(a + BLOCK, d)) for a in range(0, d, BLOCK)]
        amax = torch.stack([x[:, a:b].abs().max(1).values for a, b in edges], 1)
        out["scales"] = torch.where(amax == 0, torch.ones_like(amax), amax / 127)
        wide = torch.cat([out["scales"][:, i:i + 1].expand(n, b - a) for i, (a, b) in enumerate(edges)], 1)
        ratio = x / wide
        out["restored"] = torch.sign(ratio) * torch.floor(ratio.abs() + 0.5) * wide
        return out
    place = torch.arange(d, device="cuda") // BLOCK
    x = s["codes"].double() * s["scales"].double()[:, place]
    if case["op"] == "back":
        x.requires_grad_(True)
        gain.requires_grad_(True)
        (norm(x) * gain * s["dy"].double()).sum().backward()
        dx = x.grad
        if s["d_residual"] is not None:
            dx = dx + s["d_residual"].double()
        return {"dx": dx, "d_weight": gain.grad}
    if case["norm"]:
        x = norm(x) * gain
    return {"d_weight": torch.einsum("ti,tj->ij", s["dy"].double(), x)}
