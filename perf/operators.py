"""Cases, plain forms and exact values of the fine-tuning step's operators.

Three groups of operators stand around the adapted linears in a training step:
the normalisation in front of them (layer norm / RMS norm), the token log
probabilities behind the output projection, and AdamW over the adapter tensors.
``run`` computes them with elementary torch operations in 32 bits, or, where
``own`` is true, through ``dorafactors_b200``; ``exact`` computes them from
their definitions in 64 bits.

The 8-bit moments of AdamW are small floating-point numbers with one scale for
each block of 256 elements of a parameter (the last block may be short):

  first moment   sign, 4 exponent and 3 mantissa bits: code c of 1..127 stands for
                 2^(c // 8 - 15) * (1 + c % 8 / 8), code 0 for zero, rounded to nearest
  second moment  5 exponent and 3 mantissa bits: code c of 1..255 stands for
                 2^(c // 8 - 31) * (1 + c % 8 / 8), code 0 for zero; rounded up or down
                 by 16 bits from a hash of (seed, step, parameter, element), so that
                 the small changes of a slow average are kept in the mean

each times the block's scale, which is its largest magnitude / 1.875.
"""

import math

import torch

own = False

BLOCK = 256  # elements that share a scale, and the granule of the flat buffers
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
LR, BETAS, EPS, DECAY, SEED = 2e-4, (0.9, 0.999), 1e-8, 0.01, 17
PROJECTIONS = ("q", "k", "v", "o", "gate", "up", "down")


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    """The path's work at its real sizes: widths and token counts of the repository's layer and model configurations."""
    return [
        # One token of a decode step in front of a 4096-wide projection: latency.
        {"name": "rms-forward-1x4096", "op": "norm", "kind": "rms", "pass": "forward", "rows": 1, "cols": 4096,
         "dtype": "bfloat16", "wdtype": "bfloat16", "gap": 0},
        # The activations in front of the high-rank layer: 16384 tokens, 8192 wide.
        {"name": "layer-forward-16384x8192", "op": "norm", "kind": "layer", "pass": "forward", "rows": 16384,
         "cols": 8192, "dtype": "bfloat16", "wdtype": "bfloat16", "gap": 0},
        # The model configuration's batch of 8 x 4096 tokens, the norm's weight trained in fp32.
        {"name": "rms-backward-32768x4096", "op": "norm", "kind": "rms", "pass": "backward", "rows": 32768,
         "cols": 4096, "dtype": "bfloat16", "wdtype": "float32", "gap": 0},
        # The same for the wide layer, with mean, weight and bias.
        {"name": "layer-backward-16384x8192", "op": "norm", "kind": "layer", "pass": "backward", "rows": 16384,
         "cols": 8192, "dtype": "bfloat16", "wdtype": "bfloat16", "gap": 0},
        # fp32, rows and columns of no round size, forward and backward through autograd.
        {"name": "layer-train-1021x5003-fp32", "op": "norm", "kind": "layer", "pass": "train", "rows": 1021,
         "cols": 5003, "dtype": "float32", "wdtype": "float32", "gap": 0},
        # One sampled token of one sequence with its 20 best alternatives, a tenth of the vocabulary banned.
        {"name": "logprobs-decode-1x128256", "op": "logprobs", "pass": "forward", "rows": 1, "vocab": 128256,
         "dtype": "bfloat16", "top_k": 20, "entropy": True, "temperature": 1.0, "gap": 0, "banned": 0.1,
         "ignored": 0.0},
        # Scoring a short answer with a vocabulary of odd size in fp32, five alternatives a token.
        {"name": "logprobs-score-48x32003-fp32", "op": "logprobs", "pass": "forward", "rows": 48, "vocab": 32003,
         "dtype": "float32", "top_k": 5, "entropy": False, "temperature": 0.7, "gap": 0, "banned": 0.0,
         "ignored": 0.0},
        # One 4096-token sequence of a training step, the prompt's tokens ignored.
        {"name": "logprobs-forward-4096x128256", "op": "logprobs", "pass": "forward", "rows": 4096, "vocab": 128256,
         "dtype": "bfloat16", "top_k": 0, "entropy": True, "temperature": 1.0, "gap": 0, "banned": 0.0,
         "ignored": 0.1},
        # Its gradient with an entropy term.
        {"name": "logprobs-backward-4096x128256", "op": "logprobs", "pass": "backward", "rows": 4096, "vocab": 128256,
         "dtype": "bfloat16", "top_k": 0, "entropy": True, "temperature": 1.0, "gap": 0, "banned": 0.0,
         "ignored": 0.1},
        # One adapted 4096 x 4096 layer, r = 16: A, B and the magnitude, 135168 elements.
        {"name": "adamw-layer-r16", "op": "adamw", "layers": 1, "projections": 1, "hidden": 4096, "ffn": 14336,
         "kv": 1024, "rank": 16, "dtype": "float32", "bits": 32, "master": False, "step": 3},
        # Every adapter of the 32-layer model configuration, r = 128: 672 tensors, 337M elements, fp32.
        {"name": "adamw-model-r128-fp32", "op": "adamw", "layers": 32, "projections": 7, "hidden": 4096, "ffn": 14336,
         "kv": 1024, "rank": 128, "dtype": "float32", "bits": 32, "master": False, "step": 100},
        # The same adapters in bf16 with moments in 8 bits.
        {"name": "adamw-model-r128-8bit", "op": "adamw", "layers": 32, "projections": 7, "hidden": 4096, "ffn": 14336,
         "kv": 1024, "rank": 128, "dtype": "bfloat16", "bits": 8, "master": False, "step": 100},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: sizes spread over their logarithm, odd ones among them."""
    op = rng.choice(("norm", "logprobs", "adamw"))
    if op == "norm":
        cols = _log_int(rng, 64, 28672)
        cols = cols if rng.random() < 0.4 else max(8, cols // 8 * 8)
        rows = _log_int(rng, 1, max(1, min(32768, 16384 * 8192 // cols)))
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
        if dtype == "float32":
            rows = max(1, rows // 2)
        return {"op": op, "kind": rng.choice(("layer", "rms")), "pass": rng.choice(("forward", "backward", "train")),
                "rows": rows, "cols": cols, "dtype": dtype, "wdtype": rng.choice((dtype, "float32")),
                "gap": rng.choice((0, 0, 8, 5))}
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 128256)
        vocab = vocab if rng.random() < 0.5 else vocab // 64 * 64
        what = rng.choice(("forward", "forward", "backward", "train"))
        top_k = rng.choice((0, 1, 5, 20)) if what == "forward" else 0
        most = (1 << 25 if top_k else 1 << 28) // vocab
        return {"op": op, "pass": what, "rows": _log_int(rng, 1, max(1, min(4096, most))), "vocab": vocab,
                "dtype": rng.choice(("bfloat16", "bfloat16", "float16", "float32")), "top_k": top_k,
                "entropy": rng.random() < 0.5, "temperature": rng.choice((1.0, 0.7, 1.3)),
                "gap": rng.choice((0, 0, 61, 64)), "banned": rng.choice((0.0, 0.1)), "ignored": rng.choice((0.0, 0.1))}
    hidden = _log_int(rng, 256, 4096)
    hidden = hidden if rng.random() < 0.3 else hidden // 64 * 64
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    return {"op": op, "layers": _log_int(rng, 1, 24), "projections": rng.choice((1, 4, 7)), "hidden": hidden,
            "ffn": hidden * 7 // 2, "kv": hidden // 4, "rank": _log_int(rng, 4, 128), "dtype": dtype,
            "bits": rng.choice((32, 8)), "master": dtype != "float32" and rng.random() < 0.5,
            "step": rng.choice((0, 10, 1000))}


def work(case):
    """Bytes that have to move once, and operations, of one pass."""
    if case["op"] == "norm":
        n, c, r = case["rows"] * case["cols"], case["cols"], case["rows"]
        e, w = _size(case["dtype"]), _size(case["wdtype"])
        layer = case["kind"] == "layer"
        vectors = c * w * (2 if layer else 1)  # weight and, for a layer norm, bias
        stats = 4 * r * (2 if layer else 1)
        forward = {"bytes": 2 * e * n + vectors + stats, "flops": 8 * n}
        backward = {"bytes": 3 * e * n + c * w + vectors + stats, "flops": 14 * n}
        if case["pass"] == "train":  # x and the statistics are needed again by the backward pass
            return {k: forward[k] + backward[k] for k in forward}
        return forward if case["pass"] == "forward" else backward
    if case["op"] == "logprobs":
        rows = max(1, int(round(case["rows"] * (1 - case["ignored"]))))  # ignored rows are not read
        n, e = rows * case["vocab"], _size(case["dtype"])
        forward = {"bytes": e * n + case["rows"] * (20 + 12 * case["top_k"]), "flops": (6 if case["entropy"] else 4) * n}
        backward = {"bytes": e * n + e * case["rows"] * case["vocab"] + 28 * case["rows"], "flops": 6 * n}
        if case["pass"] == "train":
            return {k: forward[k] + backward[k] for k in forward}
        return forward if case["pass"] == "forward" else backward
    n, e = sum(_numel(s) for s in _shapes(case)), _size(case["dtype"])
    per = 3 * e + (8 if case["master"] else 0)  # parameter and gradient in, parameter out
    # Moments in and out; those of 8 bits come back as the values that they stand for, too.
    per += 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return {"bytes": per * n, "flops": 14 * n}


def _size(dtype):
    return 4 if dtype == "float32" else 2


def _numel(shape):
    return shape[0] * (shape[1] if len(shape) > 1 else 1)


def _shapes(case):
    """A, B and the magnitude of each adapted projection, layer by layer."""
    h, f, kv, r = case["hidden"], case["ffn"], case["kv"], case["rank"]
    out_in = {"q": (h, h), "k": (kv, h), "v": (kv, h), "o": (h, h), "gate": (f, h), "up": (f, h), "down": (h, f)}
    one = []
    for name in PROJECTIONS[: case["projections"]]:
        out, inp = out_in[name]
        one += [(r, inp), (out, r), (out,)]
    return one * case["layers"]


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _rows(values, dtype, gap):
    """``values`` rounded to ``dtype``, as rows of a wider buffer where ``gap`` is not zero."""
    if not gap:
        return values.to(dtype)
    wide = torch.full((values.shape[0], values.shape[1] + gap), float("nan"), device="cuda", dtype=dtype)
    wide[:, : values.shape[1]] = values
    return wide[:, : values.shape[1]]


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "norm":
        rows, cols, dt, wdt = case["rows"], case["cols"], DTYPES[case["dtype"]], DTYPES[case["wdtype"]]
        # Residual-stream activations: per-channel scales and a non-zero mean.
        s["x"] = _rows(_randn(g, rows, cols) * (0.5 + _randn(g, cols).abs()) + 0.3, dt, case["gap"])
        s["weight"] = (1 + 0.2 * _randn(g, cols)).to(wdt)
        s["bias"] = (0.1 * _randn(g, cols)).to(wdt) if case["kind"] == "layer" else None
        s["eps"] = 1e-5
        if case["pass"] != "forward":
            s["dy"] = _rows(_randn(g, rows, cols), dt, case["gap"])
        if case["pass"] == "backward":
            _, s["mean"], s["rstd"] = _norm_forward(s)
        if case["pass"] == "train":
            s["params"] = [t.requires_grad_() for t in (s["x"], s["weight"], s["bias"]) if t is not None]
    elif case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = _randn(g, rows, vocab) * 2.5
        targets = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
        # Most tokens are likely ones: their logit stands out by 2 to 20.
        lift = 2 + 18 * torch.rand(rows, device="cuda", generator=g)
        x[torch.arange(rows, device="cuda"), targets] += lift * (torch.rand(rows, device="cuda", generator=g) < 0.8)
        if case["banned"]:
            banned = torch.rand(vocab, device="cuda", generator=g) < case["banned"]
            banned[0] = False
            keep = x.gather(1, targets[:, None])
            x.masked_fill_(banned, -math.inf)
            x.scatter_(1, targets[:, None], keep)
        if case["ignored"]:
            targets[: int(round(rows * case["ignored"]))] = -100
        s["logits"], s["targets"] = _rows(x, DTYPES[case["dtype"]], case["gap"]), targets
        if case["pass"] == "train":
            s["logits"] = s["logits"].requires_grad_()
        if case["pass"] != "forward":
            s["g_logprobs"] = -(0.5 + torch.rand(rows, device="cuda", generator=g)) / rows
            s["g_entropy"] = -0.01 * torch.rand(rows, device="cuda", generator=g) / rows if case["entropy"] else None
        if case["pass"] == "backward":
            r = _logprobs_forward(s)
            s["lse"], s["entropies"] = r["logsumexp"], r.get("entropy")
    else:
        _prepare_adamw(case, s, g)
    return s


def _prepare_adamw(case, s, g):
    """Parameters and gradients are views of flat buffers, each at a multiple of 256 elements; moments alike."""
    shapes, dt = _shapes(case), DTYPES[case["dtype"]]
    sizes = [_numel(x) for x in shapes]
    blocks = [-(-n // BLOCK) for n in sizes]
    starts = [0]
    for b in blocks:
        starts.append(starts[-1] + b * BLOCK)
    total = starts.pop()

    lens = torch.tensor(sizes, device="cuda")
    nblocks = torch.tensor(blocks, device="cuda")
    tensor = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), nblocks)  # of each block
    first = torch.cumsum(nblocks, 0) - nblocks
    within = torch.arange(total // BLOCK, device="cuda") - first[tensor]  # block's number in its tensor
    live = (within[:, None] * BLOCK + torch.arange(BLOCK, device="cuda") < lens[tensor][:, None]).reshape(-1)

    # Gradients of an adapter differ by orders of magnitude from tensor to tensor and from element to element.
    size = torch.exp(_randn(g, len(sizes)) * 2 - 9)[tensor].repeat_interleave(BLOCK) * torch.exp(_randn(g, total))
    s["p"] = (_randn(g, total) * 0.02 * live).to(dt)
    s["g"] = (_randn(g, total) * size * live).to(dt)
    zero = case["step"] == 0
    m = torch.zeros(total, device="cuda") if zero else _randn(g, total) * size * 0.3 * live
    v = torch.zeros(total, device="cuda") if zero else (size * size * (0.5 + torch.rand(total, device="cuda", generator=g))) * live
    s["tensor"], s["within"] = tensor, within
    s["sizes"], s["starts"] = sizes, starts
    s["master"] = s["p"].float() * (1 + 1e-3 * _randn(g, total)) if case["master"] else None
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["m_scale"] = _encode_signed(m)
        s["v"], s["v_scale"] = _encode_unsigned(v, torch.full((total // BLOCK, BLOCK), 1 << 19, device="cuda", dtype=torch.int32))
    s["t"] = case["step"]
    if own:  # the optimizer that a program keeps, its moments loaded as from a checkpoint
        from dorafactors_b200.optim import AdamW

        views = [s["p"][a: a + n].view(shape) for a, n, shape in zip(starts, sizes, shapes)]
        params = [torch.nn.Parameter(x) for x in views]
        for p, a, n in zip(params, starts, sizes):
            p.grad = s["g"][a: a + n].view(p.shape)
        opt = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                    master_weights=case["master"], seed=SEED)
        saved = opt.state_dict()
        for i, (p, a, n) in enumerate(zip(params, starts, sizes)):
            st = {"step": case["step"]}
            part, of = slice(a, a + n), slice(a // BLOCK, a // BLOCK + -(-n // BLOCK))
            if case["bits"] == 32:
                st["exp_avg"], st["exp_avg_sq"] = s["m"][part].view(p.shape), s["v"][part].view(p.shape)
            else:
                st["exp_avg_codes"], st["exp_avg_scale"] = s["m"][part].view(p.shape), s["m_scale"][of]
                st["exp_avg_sq_codes"], st["exp_avg_sq_scale"] = s["v"][part].view(p.shape), s["v_scale"][of]
            if case["master"]:
                st["master"] = s["master"][part].view(p.shape)
            saved["state"][i] = st
        opt.load_state_dict(saved)
        s["optimizer"] = opt
        for name in ("m", "v", "m_scale", "v_scale", "master"):  # the optimizer holds them now
            s.pop(name, None)


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(s):
    return {"norm": _run_norm, "logprobs": _run_logprobs, "adamw": _run_adamw}[s["op"]](s)


def _run_norm(s):
    if own:
        from dorafactors_b200 import norms

        layer = s["kind"] == "layer"
        if s["pass"] == "forward":
            if layer:
                return norms.layer_norm_forward(s["x"], s["weight"], s["bias"], s["eps"])
            return norms.rms_norm_forward(s["x"], s["weight"], s["eps"])
        if s["pass"] == "backward":
            if layer:
                return norms.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
            return norms.rms_norm_backward(s["dy"], s["x"], s["weight"], s["rstd"])
        y = norms.layer_norm(s["x"], s["weight"], s["bias"], s["eps"]) if layer else norms.rms_norm(s["x"], s["weight"], s["eps"])
        return (y, *torch.autograd.grad(y, s["params"], s["dy"]))
    with torch.no_grad():
        if s["pass"] == "forward":
            y, mean, rstd = _norm_forward(s)
            return (y, mean, rstd) if s["kind"] == "layer" else (y, rstd)
        if s["pass"] == "backward":
            return _norm_backward(s, s["mean"], s["rstd"])
        y, mean, rstd = _norm_forward(s)
        return (y, *_norm_backward(s, mean, rstd))


def _norm_forward(s):
    x = s["x"].detach().float()
    mean = None
    if s["kind"] == "layer":
        mean = x.sum(1) * (1 / x.shape[1])
        x = x - mean[:, None]
    rstd = ((x * x).sum(1) * (1 / x.shape[1]) + s["eps"]).rsqrt()
    y = x * rstd[:, None] * s["weight"].detach().float()
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    return y.to(s["x"].dtype), mean, rstd


def _norm_backward(s, mean, rstd):
    dy, x, w = s["dy"].float(), s["x"].detach().float(), s["weight"].detach().float()
    layer = s["kind"] == "layer"
    xh = (x - mean[:, None]) * rstd[:, None] if layer else x * rstd[:, None]
    a = dy * w
    dx = a - xh * ((a * xh).sum(1, keepdim=True) * (1 / x.shape[1]))
    if layer:
        dx = dx - a.sum(1, keepdim=True) * (1 / x.shape[1])
    dx = (dx * rstd[:, None]).to(s["x"].dtype)
    dw = (dy * xh).sum(0).to(s["weight"].dtype)
    return (dx, dw, dy.sum(0).to(s["weight"].dtype)) if layer else (dx, dw)


def _run_logprobs(s):
    if own:
        from dorafactors_b200 import logprobs

        if s["pass"] == "backward":
            return logprobs.token_logprobs_backward(s["g_logprobs"], s["g_entropy"], None, s["logits"], s["targets"],
                                                    s["lse"], s["entropies"], temperature=s["temperature"])
        r = logprobs.token_logprobs(s["logits"], s["targets"], temperature=s["temperature"], entropy=s["entropy"],
                                    top_k=s["top_k"])
        out = {"logprobs": r.logprobs, "logsumexp": r.logsumexp}
        if s["entropy"]:
            out["entropy"] = r.entropy
        if s["top_k"]:
            out["top_logprobs"], out["top_indices"] = r.top_logprobs, r.top_indices
        if s["pass"] == "train":
            ys, gs = [r.logprobs], [s["g_logprobs"]]
            if s["entropy"]:
                ys, gs = ys + [r.entropy], gs + [s["g_entropy"]]
            out["grad"] = torch.autograd.grad(ys, s["logits"], gs)[0]
            out = {k: t.detach() for k, t in out.items()}
        return out
    with torch.no_grad():
        if s["pass"] == "backward":
            return _logprobs_backward(s, s["lse"], s["entropies"])
        out = _logprobs_forward(s)
        if s["pass"] == "train":
            out["grad"] = _logprobs_backward(s, out["logsumexp"], out.get("entropy"))
        return out


def _logprobs_forward(s):
    x = s["logits"].detach().float() * (1 / s["temperature"])
    used = s["targets"] != -100
    top = x.max(1, keepdim=True).values
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    lse = top + total.log()
    given = x.gather(1, s["targets"].clamp(min=0)[:, None])
    out = {"logprobs": torch.where(used, (given - lse)[:, 0], 0.0), "logsumexp": torch.where(used, lse[:, 0], 0.0)}
    if s["entropy"]:
        p = e / total
        logp = torch.where(p > 0, x - lse, 0.0)
        out["entropy"] = torch.where(used, -(p * logp).sum(1), 0.0)
    if s["top_k"]:
        values, at = x.sort(dim=1, descending=True, stable=True)
        k = s["top_k"]
        out["top_logprobs"] = torch.where(used[:, None], values[:, :k] - lse, 0.0)
        out["top_indices"] = torch.where(used[:, None], at[:, :k], -1)
    return out


def _logprobs_backward(s, lse, entropies):
    x = s["logits"].detach().float() * (1 / s["temperature"])
    used = s["targets"] != -100
    logp = x - lse[:, None]
    p = logp.exp()
    d = -s["g_logprobs"][:, None] * p
    if s["entropy"]:
        d = d - s["g_entropy"][:, None] * p * torch.where(p > 0, logp + entropies[:, None], 0.0)
    d = d.scatter_add(1, s["targets"].clamp(min=0)[:, None], s["g_logprobs"][:, None])
    d = torch.where(used[:, None], d * (1 / s["temperature"]), 0.0)
    return d.to(s["logits"].dtype)


def _run_adamw(s):
    if own:
        opt = s["optimizer"]
        opt.step()
        m, v = opt.moments()
        out = {"p": s["p"], "exp_avg": m, "exp_avg_sq": v}
        if s["op"] == "adamw" and opt.param_groups[0]["master_weights"]:
            out["master"] = opt.masters()
        return out
    with torch.no_grad():
        return _adamw(s)


def _adamw(s):
    s["t"] += 1
    (b1, b2), t = BETAS, s["t"]
    g = s["g"].float()
    p = s["p"].float() if s["master"] is None else s["master"]
    m, v = s["m"], s["v"]
    if s["bits"] == 8:
        m, v = _decode_signed(m, s["m_scale"]), _decode_unsigned(v, s["v_scale"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    denom = v.sqrt() * (1 / math.sqrt(1 - b2**t)) + EPS
    p = p * (1 - LR * DECAY) - (m / denom) * (LR / (1 - b1**t))
    if s["master"] is not None:
        s["master"].copy_(p)
    s["p"].copy_(p)
    if s["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        out = {"p": s["p"], "exp_avg": s["m"], "exp_avg_sq": s["v"]}
    else:
        s["m"], s["m_scale"] = _encode_signed(m)
        s["v"], s["v_scale"] = _encode_unsigned(v, _dither(s, t) << 4)
        out = {"p": s["p"], "exp_avg": _decode_signed(s["m"], s["m_scale"]),
               "exp_avg_sq": _decode_unsigned(s["v"], s["v_scale"])}
    if s["master"] is not None:
        out["master"] = s["master"]
    return out


# 8-bit moments.  Codes are the upper bits of the fp32 number, so that rounding is an integer addition.
def _block_scale(x):
    top = x.abs().view(-1, BLOCK).max(1).values
    live = top >= 2.0**-100  # below it the whole block counts as zero
    inverse = torch.where(live, torch.full_like(top, 1.875) / top, 0.0)
    return torch.where(live, top * (8 / 15), 0.0), inverse


def _encode_signed(m):
    scale, inverse = _block_scale(m)
    y = (m.abs().view(-1, BLOCK) * inverse[:, None]).view(torch.int32)
    code = (((y + (1 << 19)) >> 20) - (112 << 3)).clamp(0, 127)
    return (code + 128 * (m.view(-1, BLOCK) < 0)).to(torch.uint8).view(-1), scale


def _decode_signed(code, scale):
    c = code.view(-1, BLOCK).to(torch.int32)
    u = torch.where(c & 127 > 0, (((c & 127) + (112 << 3)) << 20).view(torch.float32), 0.0)
    return (torch.where(c > 127, -u, u) * scale[:, None]).view(-1)


def _encode_unsigned(v, tail):
    scale, inverse = _block_scale(v)
    y = (v.view(-1, BLOCK) * inverse[:, None]).view(torch.int32)
    code = torch.where(v.view(-1, BLOCK) > 0, (((y + tail) >> 20) - (96 << 3)).clamp(1, 255), 0)
    return code.to(torch.uint8).view(-1), scale


def _decode_unsigned(code, scale):
    c = code.view(-1, BLOCK).to(torch.int32)
    u = torch.where(c > 0, ((c + (96 << 3)) << 20).view(torch.float32), 0.0)
    return (u * scale[:, None]).view(-1)


def _dither(s, t):
    """16 bits for each element: a 32-bit hash of (seed, step, parameter, pair of elements), its halves for the two."""
    low = 0xFFFFFFFF
    key = (SEED + t * 0x9E3779B1 + s["tensor"] * 0xC2B2AE35) & low
    x = ((s["within"] * (BLOCK // 2))[:, None] + torch.arange(BLOCK // 2, device="cuda")) * 0x85EBCA77 + key[:, None]
    x = x & low
    x = ((x ^ (x >> 15)) * 0xA2C79B4D) & low
    x = ((x ^ (x >> 13)) * 0x5BD0E6A7) & low
    x = x ^ (x >> 16)
    return torch.stack((x & 0xFFFF, x >> 16), -1).view(-1, BLOCK).to(torch.int32)


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    return {"norm": _exact_norm, "logprobs": _exact_logprobs, "adamw": _exact_adamw}[case["op"]](case, seed)


@torch.no_grad()
def _exact_norm(case, seed):
    s = prepare(case, seed)
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    rms = case["kind"] == "rms"
    mean = torch.zeros(len(x), device="cuda", dtype=torch.float64) if rms else x.mean(1)
    std = torch.sqrt(torch.mean((x - mean[:, None]) ** 2, 1) + s["eps"])
    xh = (x - mean[:, None]) / std[:, None]
    stats = [1 / std] if rms else [mean, 1 / std]
    y = xh * w if rms else xh * w + s["bias"].detach().double()
    if case["pass"] == "forward":
        return [y, *stats]
    dy = s["dy"].double()
    a = dy * w
    dx = (a - torch.mean(a * xh, 1)[:, None] * xh - (0 if rms else torch.mean(a, 1)[:, None])) / std[:, None]
    grads = [dx, torch.sum(dy * xh, 0)] + ([] if rms else [torch.sum(dy, 0)])
    return grads if case["pass"] == "backward" else [y, *grads]


@torch.no_grad()
def _exact_logprobs(case, seed):
    s = prepare(case, seed)
    t, used = s["targets"].clamp(min=0)[:, None], s["targets"] >= 0
    logp = s["logits"].detach().double() / case["temperature"]
    lse = torch.logsumexp(logp, 1)
    logp -= lse[:, None]
    p = logp.exp()
    out = {"logprobs": logp.gather(1, t)[:, 0] * used, "logsumexp": lse * used}
    h = -torch.special.xlogy(p, p).sum(1)
    if case["entropy"]:
        out["entropy"] = h * used
    if case["top_k"]:
        out["top_logprobs"], out["top_indices"] = logp.topk(case["top_k"]).values * used[:, None], None
    if case["pass"] == "forward":
        return out
    gl = s["g_logprobs"].double()
    d = -gl[:, None] * p
    if case["entropy"]:
        d -= s["g_entropy"].double()[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
    d.scatter_add_(1, t, gl[:, None])
    d = d * used[:, None] / case["temperature"]
    if case["pass"] == "backward":
        return d
    return {**out, "grad": d}


@torch.no_grad()
def _exact_adamw(case, seed):
    global own
    kept, own = own, False
    s = prepare(case, seed)
    own = kept
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m, v = _stands_for(s["m"], s["m_scale"], True), _stands_for(s["v"], s["v_scale"], False)
    t, g = case["step"] + 1, s["g"].double()
    p = (s["p"] if s["master"] is None else s["master"]).double()
    m += (1 - BETAS[0]) * (g - m)
    v += (1 - BETAS[1]) * (g * g - v)
    p = p - LR * DECAY * p - LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
    out = {"p": p, "exp_avg": m, "exp_avg_sq": v}
    if case["bits"] == 8:
        half = torch.full((1, 1), 0.5, device="cuda", dtype=torch.float64)
        out["exp_avg"] = _rounded(m, half, 15, 127)
        out["exp_avg_sq"] = _rounded(v, _dither(s, t).double() / 65536, 31, 255)
    if s["master"] is not None:
        out["master"] = p
    return out


def _stands_for(code, scale, signed):
    c = code.view(-1, BLOCK).double()
    sign = torch.where(c > 127, -1.0, 1.0) if signed else 1.0
    c = c % 128 if signed else c
    u = torch.exp2(torch.floor(c / 8) - (15 if signed else 31)) * (1 + c % 8 / 8)
    return (sign * torch.where(c > 0, u, 0.0) * scale.double()[:, None]).view(-1)


def _rounded(x, up, lowest, most):
    """The value of the code that x has in its block of 256; ``up`` of the distance to the next code rounds upwards."""
    x = x.view(-1, BLOCK)
    top = x.abs().max(1, keepdim=True).values
    fraction, power = torch.frexp(x.abs() / torch.where(top > 0, top, 1.0) * 1.875)
    at = torch.floor((power.double() - 1 + lowest + (2 * fraction - 1)) * 8 + up)  # codes are even within a power of two
    at = at.clamp(0 if most == 127 else 1, most)
    u = torch.where((at > 0) & (x != 0), torch.exp2(torch.floor(at / 8) - lowest) * (1 + at % 8 / 8), 0.0)
    return (x.sign() * u * top / 1.875).view(-1)
