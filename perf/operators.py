"""Cases and plain forms of the operators around the NVFP4 linears of a feed-forward sublayer.

Five operators, each as its formula in elementary torch operations (``own`` false) and as the call a
user makes of ``radiance_b200.nvfp4`` (``own`` true):

* ``mm``: the block-scaled product with bias, activation, dropout and residual in its epilogue,
  ``y = residual + drop(act(ga gb A B^T + bias))``;
* ``mm_grad``: the backward of that epilogue, ``dz = drop(dy) act'(z)`` with the global scale of dz
  and the bias gradient;
* ``dropout``: counter-based dropout with an optional residual, forward and backward;
* ``route``: top-k routing of tokens to experts with per-expert counts, row plan and balance loss,
  and the gradient of the router logits;
* ``rows``: moving tokens to their experts' rows and the weighted sum back, and the gradients.
"""

import math

import numpy as np
import torch

own = False

ACTIVATIONS = ("none", "relu", "relu2", "silu", "gelu", "gelu_tanh")
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------


def listed():
    return [
        # A dense block's down projection over a batch of 16384 tokens: bias, dropout and the
        # residual stream added in the epilogue.
        dict(name="mm down 16384", op="mm", m=16384, n=2048, k=5632, act="none", p=0.1, bias=True, residual=True,
             preact=False, dtype="bf16"),
        # A plain (ungated) up projection of the same block in training: GELU, with the
        # pre-activations kept for the backward pass.
        dict(name="mm up 16384", op="mm", m=16384, n=5632, k=2048, act="gelu", p=0.0, bias=True, residual=False,
             preact=True, dtype="bf16"),
        # A small fp32 layer whose sizes are no multiple of the tiles (128-row and 128-column tails,
        # a short last contraction step): latency counts.
        dict(name="mm small fp32", op="mm", m=384, n=640, k=1088, act="relu2", p=0.2, bias=True, residual=True,
             preact=True, dtype="fp32"),
        # The backward pass of that up projection's epilogue: gradient, its global scale, bias gradient.
        dict(name="mm_grad up 16384", op="mm_grad", rows=16384, cols=5632, act="gelu", p=0.0, bias=True,
             dtype="bf16"),
        # A small fp32 layer's, with dropout.
        dict(name="mm_grad small fp32", op="mm_grad", rows=640, cols=1152, act="silu", p=0.1, bias=True,
             dtype="fp32"),
        # Residual dropout of a block's output in training, forward and backward.
        dict(name="dropout 16384", op="dropout", rows=16384, cols=2048, p=0.1, residual=True, train=True,
             dtype="bf16"),
        # The smallest: a few odd rows in fp32, no residual.
        dict(name="dropout tiny fp32", op="dropout", rows=37, cols=129, p=0.25, residual=False, train=False,
             dtype="fp32"),
        # The router of an 8-expert layer, top 2 of 16384 tokens, in training.
        dict(name="route 16384x8", op="route", tokens=16384, experts=8, k=2, renorm=True, bias=False, padded=False,
             dtype="fp32"),
        # Many small experts, a selection bias, softmax weights as they are, and a padded batch.
        dict(name="route 4099x160", op="route", tokens=4099, experts=160, k=6, renorm=False, bias=True, padded=True,
             dtype="bf16"),
        # That 8-expert layer's rows: out to the experts and back, forward.
        dict(name="rows 16384", op="rows", tokens=16384, d=2048, experts=8, k=2, residual=True, train=False,
             dtype="bf16"),
        # The same in training: forward and all gradients.
        dict(name="rows train 16384", op="rows", tokens=16384, d=2048, experts=8, k=2, residual=True, train=True,
             dtype="bf16"),
        # A few tokens over many experts, as when a short prompt is evaluated.
        dict(name="rows 33 tokens", op="rows", tokens=33, d=1408, experts=16, k=4, residual=False, train=False,
             dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("mm", "mm", "mm_grad", "dropout", "route", "rows"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    p = rng.choice((0.0, 0.05, 0.1, 0.2, 0.5))
    act = rng.choice(ACTIVATIONS)
    if op == "mm":
        while True:
            m, n, k = 128 * _log(rng, 1, 128), 128 * _log(rng, 1, 44), 64 * _log(rng, 1, 88)
            if m * n * k <= 16384 * 2048 * 5632 and m * n <= 16384 * 2816:
                break
        return dict(op=op, m=m, n=n, k=k, act=act, p=p, bias=rng.random() < 0.7, residual=rng.random() < 0.6,
                    preact=rng.random() < 0.4, dtype=dtype)
    if op == "mm_grad":
        while True:
            rows, cols = _log(rng, 1, 16384), _log(rng, 8, 5632)
            if rows * cols <= 16384 * 2816:
                break
        return dict(op=op, rows=rows, cols=cols, act=act, p=p, bias=rng.random() < 0.7, dtype=dtype)
    if op == "dropout":
        return dict(op=op, rows=_log(rng, 1, 16384), cols=_log(rng, 1, 2048), p=max(p, 0.05),
                    residual=rng.random() < 0.5, train=rng.random() < 0.5, dtype=dtype)
    if op == "route":
        experts = _log(rng, 2, 256)
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=experts, k=rng.randint(1, min(8, experts)),
                    renorm=rng.random() < 0.5, bias=rng.random() < 0.5, padded=rng.random() < 0.5, dtype=dtype)
    experts = _log(rng, 2, 64)
    k = rng.randint(1, min(4, experts))
    while True:
        tokens, d = _log(rng, 1, 16384), _log(rng, 8, 2048)
        if _row_bound(tokens, k, experts) * d <= 16384 * 2048:
            break
    return dict(op=op, tokens=tokens, d=d, experts=experts, k=k, residual=rng.random() < 0.5,
                train=rng.random() < 0.5, dtype=dtype)


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------


def _quantized(x):
    """(packed codes, swizzled block scales, global scale) of x (rows % 128 == 0, cols % 64 == 0):
    e2m1 codes and e4m3 scales of 16-element blocks, rounded to nearest."""
    rows, cols = x.shape
    gs = (x.abs().max() / 2688.0).clamp_min(1e-12)
    blocks = x.view(rows, cols // 16, 16)
    scale = (blocks.abs().amax(-1) / (6.0 * gs)).clamp(max=448.0).to(torch.float8_e4m3fn)
    q = blocks / (scale.float() * gs).clamp_min(1e-30).unsqueeze(-1)
    edges = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=x.device)
    code = (torch.bucketize(q.abs(), edges).to(torch.uint8) | ((q < 0).to(torch.uint8) << 3)).view(rows, cols)
    packed = (code[:, 1::2] << 4) | code[:, 0::2]
    tiles = scale.view(torch.uint8).view(rows // 128, 4, 32, cols // 64, 4)
    return packed.contiguous(), tiles.permute(0, 3, 2, 1, 4).reshape(-1).contiguous(), gs.reshape(())


def _row_bound(tokens, k, experts):
    """Rows of the expert-sorted layout that any routing of these sizes fits in: every expert that can
    receive a row ends its group at a multiple of 128."""
    pairs = tokens * k
    return (pairs + 127 * min(experts, pairs)) // 128 * 128


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    s = {"case": case}
    op = case["op"]
    if op in ("mm", "mm_grad", "dropout"):  # the seed that a program draws for this step's dropout
        s["seed"] = torch.tensor((seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), dtype=torch.int64, device="cuda")
    if op == "mm":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"] = _quantized(normal(m, k, dtype=torch.float32))
        s["b"] = _quantized(normal(n, k, dtype=torch.float32, std=k ** -0.5))
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
    elif op == "mm_grad":
        s["grad"] = normal(case["rows"], case["cols"], std=1e-3)
        s["z"] = None if case["act"] == "none" else normal(case["rows"], case["cols"])
    elif op == "dropout":
        s["x"] = normal(case["rows"], case["cols"]).requires_grad_(case["train"])
        s["residual"] = normal(case["rows"], case["cols"]) if case["residual"] else None
        s["grad"] = normal(case["rows"], case["cols"]) if case["train"] else None
    elif op == "route":
        t, e = case["tokens"], case["experts"]
        s["logits"] = normal(t, e)
        s["bias"] = normal(e, dtype=torch.float32, std=0.1) if case["bias"] else None
        s["valid"] = None
        if case["padded"]:  # the last eighth of the batch is padding, holding whatever was there
            s["valid"] = torch.arange(t, device="cuda") < t - t // 8
            s["logits"][t - t // 8:] = float("nan")
        s["grad_w"] = normal(t, case["k"], dtype=torch.float32, std=1e-2)
        s["grad_loss"] = torch.tensor(0.01, device="cuda")
        s["logits"].requires_grad_(True)
    else:
        t, d, e, k = case["tokens"], case["d"], case["experts"], case["k"]
        r = _route(normal(t, e, dtype=torch.float32), k, None, None, True)
        rows = _row_bound(t, k, e)
        s.update(r)
        s["num_rows"] = rows
        s["x"] = normal(t, d).requires_grad_(case["train"])
        s["y"] = normal(rows, d).requires_grad_(case["train"])
        s["weights"] = s["weights"].detach().requires_grad_(case["train"])
        s["residual"] = normal(t, d) if case["residual"] else None
        if case["train"]:
            s["grad_rows"] = normal(rows, d)
            s["grad_y"] = normal(t, d)
    return s


# ------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _dequantized(q):
    """fp32 values of an operand, without its global scale."""
    packed, scale, _ = q
    rows, cols = packed.shape[0], packed.shape[1] * 2
    table = torch.tensor(_E2M1, device=packed.device)
    val = table[torch.stack((packed & 15, packed >> 4), -1).reshape(rows, cols).int()]
    r = torch.arange(rows, device=packed.device).view(-1, 1)
    c = torch.arange(cols // 16, device=packed.device).view(1, -1)
    at = ((r // 128) * (cols // 64) + c // 4) * 512 + (r % 32) * 16 + ((r % 128) // 32) * 4 + c % 4
    return (val.view(rows, cols // 16, 16) * scale.view(torch.float8_e4m3fn)[at].float().unsqueeze(-1)).view(rows, cols)


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "relu2":
        return z.clamp_min(0).square()
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "relu2":
        return 2 * z.clamp_min(0)
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return sg * (1 + z * (1 - sg))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        th = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _threshold(p):
    """The 16-bit draws below this drop their element."""
    return int(p * 65536 + 0.5)


def _keep(n, p, seed):
    """Whether each of n elements stays: element i takes the 16-bit half i % 2 of word (i % 8) // 2 of
    Philox4x32-10 (Salmon et al., 2011) with counter (i // 8, 0) and the seed as its key."""
    low = 0xFFFFFFFF
    i = torch.arange((n + 7) // 8, dtype=torch.int64, device=seed.device)
    c0, c1, c2, c3 = i & low, i >> 32, torch.zeros_like(i), torch.zeros_like(i)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits; the sign goes with the mask below
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:n] >= _threshold(p)


def _drop(x, p, seed):
    if p == 0:
        return x
    return torch.where(_keep(x.numel(), p, seed).view_as(x), x * (65536 / (65536 - _threshold(p))), 0.0)


def _route(logits, k, bias, valid, renorm):
    """Top-k routing in fp32; ties go to the lower expert."""
    x = logits.detach().float()
    t, e = x.shape
    if valid is not None:
        x = torch.where(valid.view(-1, 1), x, 0.0)
    score = x if bias is None else x + bias
    experts = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :k]
    z = torch.exp(x - x.amax(-1, keepdim=True))
    prob = z / z.sum(-1, keepdim=True)
    weights = prob.gather(1, experts)
    if renorm:
        weights = weights / weights.sum(-1, keepdim=True)
    n = torch.tensor(t, device=x.device) if valid is None else valid.sum()
    if valid is not None:
        experts = torch.where(valid.view(-1, 1), experts, -1)
        weights = torch.where(valid.view(-1, 1), weights, 0.0)
        prob = torch.where(valid.view(-1, 1), prob, 0.0)
    flat = experts.reshape(-1)
    counts = (flat.view(-1, 1) == torch.arange(e, device=x.device)).sum(0)
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64, device=x.device), ((counts + 127) // 128 * 128).cumsum(0)))
    by_expert = torch.sort(flat, stable=True).indices  # pairs without an expert first
    place = torch.empty_like(by_expert).scatter_(0, by_expert, torch.arange(t * k, device=x.device))
    start = (flat < 0).sum() + counts.cumsum(0) - counts
    at = flat.clamp_min(0)
    rows = torch.where(flat < 0, -1, offsets[at] + place - start[at])
    share = counts.double() / counts.sum()
    loss = e * (share * prob.double().sum(0)).sum() / n
    return {"weights": weights, "experts": experts.int(), "counts": counts.long(), "offsets": offsets,
            "rows": rows.view(t, k).int(), "balance_loss": loss.float(), "prob": prob, "share": share, "routed": n}


def _route_pass(s):
    c = s["case"]
    r = _route(s["logits"], c["k"], s["bias"], s["valid"], c["renorm"])
    t, e = s["logits"].shape
    prob, w, gw = r.pop("prob"), r["weights"], s["grad_w"]
    per_prob = s["grad_loss"] * e * r.pop("share").float() / r.pop("routed")  # d loss / d prob of any token
    grad = prob * (per_prob - (prob * per_prob).sum(-1, keepdim=True))
    at = r["experts"].long().clamp_min(0)
    if c["renorm"]:
        grad = grad.scatter_add(1, at, w * (gw - (w * gw).sum(-1, keepdim=True)))
    else:
        grad = grad.scatter_add(1, at, w * gw) - prob * (w * gw).sum(-1, keepdim=True)
    if s["valid"] is not None:
        grad = torch.where(s["valid"].view(-1, 1), grad, 0.0)
    return {**r, "grad_logits": grad.to(s["logits"].dtype)}


def _rows_pass(s):
    c = s["case"]
    t, k = s["rows"].shape
    n, d = s["num_rows"], c["d"]
    at = s["rows"].long().view(-1)  # every pair has a row here
    x, y, w = s["x"].detach(), s["y"].detach(), s["weights"].detach()
    out = {"rows": torch.zeros(n, d, dtype=x.dtype, device=x.device).index_copy(0, at, x.repeat_interleave(k, 0))}
    picked = y[at].float().view(t, k, d)
    back = (picked * w.unsqueeze(-1)).sum(1)
    out["y"] = (back if s["residual"] is None else back + s["residual"].float()).to(x.dtype)
    if c["train"]:
        gy = s["grad_y"].float()
        out["grad_x"] = s["grad_rows"][at].float().view(t, k, d).sum(1).to(x.dtype)
        each = (gy.unsqueeze(1) * w.unsqueeze(-1)).to(x.dtype).view(t * k, d)
        out["grad_rows"] = torch.zeros(n, d, dtype=x.dtype, device=x.device).index_copy(0, at, each)
        out["grad_w"] = (picked * gy.unsqueeze(1)).sum(-1)
    return out


def _plain(s):
    c = s["case"]
    op = c["op"]
    dt = DTYPES[c["dtype"]]
    if op == "mm":
        z = (_dequantized(s["a"]) @ _dequantized(s["b"]).t()) * (s["a"][2] * s["b"][2])
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _drop(_act(z, c["act"]), c["p"], s["seed"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return {"y": y.to(dt), "z": z.to(dt)} if c["preact"] else {"y": y.to(dt)}
    if op == "mm_grad":
        dz = _drop(s["grad"].float(), c["p"], s["seed"])
        if s["z"] is not None:
            dz = dz * _act_grad(s["z"].float(), c["act"])
        out = {"grad_z": dz.to(dt)}
        out["scale"] = (out["grad_z"].abs().max().float() / 2688.0).clamp_min(1e-12)
        if c["bias"]:
            out["grad_bias"] = dz.sum(0, dtype=torch.float64).float()
        return out
    if op == "dropout":
        y = _drop(s["x"].detach().float(), c["p"], s["seed"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        out = {"y": y.to(dt)}
        if c["train"]:
            out["grad_x"] = _drop(s["grad"].float(), c["p"], s["seed"]).to(dt)
        return out
    return _route_pass(s) if op == "route" else _rows_pass(s)


# ------------------------------------------------------------------------------------------------
# The framework's calls
# ------------------------------------------------------------------------------------------------


def _own(s):
    import radiance_b200.nvfp4 as nv

    c = s["case"]
    op = c["op"]
    if op == "mm":
        a, b = (nv.NVFP4Tensor(q[0].view(torch.float4_e2m1fn_x2), q[1].view(torch.float8_e4m3fn), q[2])
                for q in (s["a"], s["b"]))
        y = nv.epilogue_mm(a, b, bias=s["bias"], activation=None if c["act"] == "none" else c["act"],
                           dropout_p=c["p"], seed=s["seed"], residual=s["residual"], out_dtype=DTYPES[c["dtype"]],
                           save_preact=c["preact"])
        return {"y": y[0], "z": y[1]} if c["preact"] else {"y": y}
    if op == "mm_grad":
        dz, gs, db = nv.epilogue_backward(s["grad"], s["z"], activation=None if c["act"] == "none" else c["act"],
                                          dropout_p=c["p"], seed=s["seed"], bias_grad=c["bias"])
        return {"grad_z": dz, "scale": gs, "grad_bias": db} if c["bias"] else {"grad_z": dz, "scale": gs}
    if op == "dropout":
        y = nv.dropout(s["x"], c["p"], seed=s["seed"], residual=s["residual"])
        if not c["train"]:
            return {"y": y}
        return {"y": y.detach(), "grad_x": torch.autograd.grad(y, s["x"], s["grad"])[0]}
    if op == "route":
        r = nv.route(s["logits"], c["k"], expert_bias=s["bias"], valid=s["valid"], renormalize=c["renorm"])
        (grad,) = torch.autograd.grad((r.weights, r.balance_loss), s["logits"], (s["grad_w"], s["grad_loss"]))
        return {"weights": r.weights.detach(), "experts": r.experts, "counts": r.counts, "offsets": r.offsets,
                "rows": r.rows, "balance_loss": r.balance_loss.detach(), "grad_logits": grad}
    r = nv.Routing(s["weights"], s["experts"], s["counts"], s["balance_loss"], s["offsets"], s["rows"], s["num_rows"])
    rows = nv.token_dispatch(s["x"], r)
    y = nv.token_combine(s["y"], r, residual=s["residual"])
    if not c["train"]:
        return {"rows": rows, "y": y}
    gx, gr, gw = torch.autograd.grad((rows, y), (s["x"], s["y"], s["weights"]), (s["grad_rows"], s["grad_y"]))
    return {"rows": rows.detach(), "y": y.detach(), "grad_x": gx, "grad_rows": gr, "grad_w": gw}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ------------------------------------------------------------------------------------------------
# Work
# ------------------------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    size = 2 if case["dtype"] == "bf16" else 4
    if op == "mm":
        m, n, k = case["m"], case["n"], case["k"]
        outs = 1 + case["residual"] + case["preact"]
        return {"bytes": (m + n) * k * 9 / 16 + outs * m * n * size + case["bias"] * n * size, "flops": 2 * m * n * k}
    if op == "mm_grad":
        n = case["rows"] * case["cols"]
        return {"bytes": (2 + (case["act"] != "none")) * n * size + case["bias"] * case["cols"] * 4, "flops": 8 * n}
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": (2 + case["residual"] + 2 * case["train"]) * n * size, "flops": 2 * n}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        # The logits once, their gradient once; per pair its weight, expert, row and weight gradient.
        return {"bytes": 2 * t * e * size + t * k * 16 + 24 * e, "flops": 8 * t * e}
    t, d, e, k = case["tokens"], case["d"], case["experts"], case["k"]
    rows = _row_bound(t, k, e)
    b = t * d + rows * d + t * k * d + t * d + case["residual"] * t * d  # dispatch; combine
    if case["train"]:  # grad_x of the dispatch; both gradients of the combine (its rows are read once more)
        b += t * k * d + t * d + t * d + rows * d
    return {"bytes": b * size + 8 * t * k, "flops": 2 * t * k * d * (3 if case["train"] else 1)}


# ------------------------------------------------------------------------------------------------
# 64-bit values
# ------------------------------------------------------------------------------------------------


def _exact_operand(q):
    """float64 values of an operand: the e2m1 bits decoded by their fields, the scale tiles unfolded."""
    packed, scale, gs = q
    rows, cols = packed.shape[0], packed.shape[1] * 2
    code = torch.empty(rows, cols, dtype=torch.uint8, device=packed.device)
    code[:, 0::2], code[:, 1::2] = packed & 15, packed >> 4
    exponent, mantissa = ((code >> 1) & 3).double(), (code & 1).double()
    mag = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.exp2(exponent - 1))
    mag = torch.where(code >= 8, -mag, mag)
    tiles = scale.view(torch.float8_e4m3fn).to(torch.float64).view(rows // 128, cols // 64, 32, 4, 4)
    sc = tiles.permute(0, 3, 2, 1, 4).reshape(rows, cols // 16)
    return mag * sc.repeat_interleave(16, 1) * gs.double()


def _exact_kept(shape, p, seed):
    """The kept elements, with Philox in numpy's unsigned integers."""
    n = math.prod(shape)
    key = np.uint64(int(seed))
    mask, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    g = np.arange((n + 7) // 8, dtype=np.uint64)
    x = [g & mask, g >> sh, np.zeros_like(g), np.zeros_like(g)]
    kk = [int(key & mask), int(key >> sh)]
    for _ in range(10):
        lo, hi = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(hi >> sh) ^ x[1] ^ np.uint64(kk[0]), hi & mask, (lo >> sh) ^ x[3] ^ np.uint64(kk[1]), lo & mask]
        kk = [(kk[0] + 0x9E3779B9) & 0xFFFFFFFF, (kk[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack(x, 1).astype(np.uint32).view(np.uint16).reshape(-1)[:n]  # little endian: low half first
    return torch.from_numpy(halves >= round(p * 65536)).view(shape).cuda()


def _exact_drop(x, p, seed):
    if p == 0:
        return x
    dropped = round(p * 65536) / 65536
    return x.masked_fill(~_exact_kept(tuple(x.shape), p, seed), 0.0) / (1 - dropped)


def _exact_act(z, act):
    """(value, derivative) in float64."""
    with torch.enable_grad():
        v = z.detach().requires_grad_(True)
        f = {"none": lambda u: u * 1.0, "relu": torch.relu, "relu2": lambda u: torch.relu(u) ** 2,
             "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda u: torch.nn.functional.gelu(u, approximate="tanh")}[act](v)
        (g,) = torch.autograd.grad(f.sum(), v)
    return f.detach(), g


def _exact_route(s):
    """The router from its definition in float64, the gradient by automatic differentiation of
    sum(weights * grad_w) + grad_loss * loss with the selection and the counts held fixed."""
    c = s["case"]
    t, e = s["logits"].shape
    live = torch.ones(t, dtype=torch.bool, device="cuda") if s["valid"] is None else s["valid"]
    with torch.enable_grad():
        x = torch.where(live[:, None], s["logits"].detach().double(), 0.0).requires_grad_(True)
        # The selection compares fp32 scores: the same sums in fp32 decide it.
        score = x.detach().float() if s["bias"] is None else x.detach().float() + s["bias"]
        pick = np.argsort(-score.cpu().numpy(), axis=1, kind="stable")[:, :c["k"]]
        pick = torch.from_numpy(pick.copy()).cuda()
        prob = torch.softmax(x, -1)
        w = prob.gather(1, pick)
        if c["renorm"]:
            w = w / w.sum(-1, keepdim=True)
        w = w * live[:, None]
        counts = torch.bincount(pick[live].reshape(-1), minlength=e).double()
        loss = e * ((counts / counts.sum()) * prob[live].mean(0)).sum()
        (grad,) = torch.autograd.grad((w * s["grad_w"].double()).sum() + s["grad_loss"].double() * loss, x)
    return {"weights": w.detach(), "experts": None, "counts": None, "offsets": None, "rows": None,
            "balance_loss": loss.detach(), "grad_logits": grad}


def _exact_rows(s):
    c = s["case"]
    t, k = s["rows"].shape
    n = s["num_rows"]
    at = s["rows"].long()
    hold = torch.full((n,), -1, dtype=torch.int64, device="cuda")  # the pair that each row holds
    hold[at.view(-1)] = torch.arange(t * k, device="cuda")
    used = (hold >= 0)[:, None]
    token, pair = hold.clamp_min(0) // k, hold.clamp_min(0)
    x, y, w = s["x"].detach(), s["y"].detach(), s["weights"].detach().double()
    out = {"rows": torch.where(used, x[token], 0.0)}
    acc = torch.zeros(t, c["d"], dtype=torch.float64, device="cuda")
    for j in range(k):
        acc += w[:, j:j + 1] * y[at[:, j]].double()
    out["y"] = acc if s["residual"] is None else acc + s["residual"].double()
    if c["train"]:
        gy = s["grad_y"].double()
        out["grad_x"] = sum(s["grad_rows"][at[:, j]].double() for j in range(k))
        out["grad_rows"] = torch.where(used, w.view(-1)[pair][:, None] * gy[token], 0.0)
        out["grad_w"] = torch.stack([(y[at[:, j]].double() * gy).sum(1) for j in range(k)], 1)
    return {name: v.double() for name, v in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    with torch.no_grad():
        if op == "mm":
            z = _exact_operand(s["a"]) @ _exact_operand(s["b"]).t()
            if s["bias"] is not None:
                z = z + s["bias"].double()
            y = _exact_drop(_exact_act(z, case["act"])[0], case["p"], s["seed"])
            if s["residual"] is not None:
                y = y + s["residual"].double()
            return {"y": y, "z": z} if case["preact"] else {"y": y}
        if op == "mm_grad":
            dz = _exact_drop(s["grad"].double(), case["p"], s["seed"])
            if s["z"] is not None:
                dz = dz * _exact_act(s["z"].double(), case["act"])[1]
            # The global scale is that of the gradient as it is handed on, rounded to its type.
            out = {"grad_z": dz, "scale": (dz.abs().max().to(dt).double() / 2688).clamp_min(1e-12)}
            if case["bias"]:
                out["grad_bias"] = dz.sum(0)
            return out
        if op == "dropout":
            y = _exact_drop(s["x"].detach().double(), case["p"], s["seed"])
            out = {"y": y if s["residual"] is None else y + s["residual"].double()}
            if case["train"]:
                out["grad_x"] = _exact_drop(s["grad"].double(), case["p"], s["seed"])
            return out
        return _exact_route(s) if op == "route" else _exact_rows(s)
