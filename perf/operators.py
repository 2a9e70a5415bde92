"""Cases of the training and scoring operators around the decoder's tail.

Three operators of ``training`` (the package's module), each with its backward pass:

  layer norm      fp16/bf16 rows with the residual add before it, fp32 gamma and beta
  cross entropy   of the tied token table's logits against the transcript's tokens
  distillation    T^2 KL(teacher's top logits, renormalised || student) over the same table

The vocabulary losses take the final states [n, d] and the token table [V, d]; neither
the logits nor their gradient is an input or an output.  Where ``own`` is false the
operators are computed in elementary torch operations in 32 bits.
"""

import importlib

import torch

own = False

EPS = 1e-5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100


def _norm(name, rows, cols, dtype, residual):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual}


def _loss(name, n, d, vocab, dtype, train, padding):
    return {"name": name, "op": "loss", "n": n, "d": d, "vocab": vocab, "dtype": dtype, "train": train,
            "padding": padding}


def _distill(name, n, d, vocab, dtype, train, k, temperature):
    return {"name": name, "op": "distill", "n": n, "d": d, "vocab": vocab, "dtype": dtype, "train": train, "k": k,
            "temperature": temperature}


def listed():
    return [
        # One decoder position of 20 beams (large-v3's width): latency alone.
        _norm("norm 20x1280 fp16", 20, 1280, "fp16", True),
        # One transcript window of the smallest model, first norm of the stack (nothing to add).
        _norm("norm 447x384 bf16", 447, 384, "bf16", False),
        # Eight 30 s windows of encoder states.
        _norm("norm 12000x1280 fp16", 12000, 1280, "fp16", True),
        # The encoder's largest batch: 64 windows.
        _norm("norm 96000x1280 bf16", 96000, 1280, "bf16", True),
        # Log-probabilities of one position of 20 beams: streams the token table.
        _loss("score 20x1280 fp16", 20, 1280, 51866, "fp16", False, 0.0),
        # Log-probabilities of 32 transcripts of 224 tokens.
        _loss("score 7168x1280 fp16", 7168, 1280, 51866, "fp16", False, 0.1),
        # One padded window of the smallest model, odd everywhere.
        _loss("loss 333x384 bf16", 333, 384, 51865, "bf16", True, 0.3),
        # A fine-tuning micro-batch of the small model: 16 transcripts of 224 tokens.
        _loss("loss 3584x768 bf16", 3584, 768, 51865, "bf16", True, 0.1),
        # 64 transcripts of 224 tokens at large-v3's width: the largest step.
        _loss("loss 14336x1280 fp16", 14336, 1280, 51866, "fp16", True, 0.1),
        # A few tokens against a teacher's five best: the table is streamed in each direction.
        _distill("distill 7x512 bf16", 7, 512, 51865, "bf16", True, 5, 1.0),
        # Ten windows of the medium model against 32 teacher logits, softened.
        _distill("distill 2240x1024 fp16", 2240, 1024, 51865, "fp16", True, 32, 2.0),
        # 32 transcripts of 224 tokens against 128 teacher logits.
        _distill("distill 7168x1280 bf16", 7168, 1280, 51866, "bf16", True, 128, 1.5),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "loss", "loss", "distill", "distill"])
    dtype = rng.choice(["fp16", "bf16"])
    width = rng.choice([384, 512, 768, 1024, 1280, 8 * rng.randint(48, 160)])
    if op == "norm":
        case = _norm("", _log_int(rng, 1, 96000), width, dtype, rng.random() < 0.6)
    else:
        vocab = rng.choice([51864, 51865, 51866, _log_int(rng, 1000, 51866)])
        train = rng.random() < 0.7
        if op == "loss":
            case = _loss("", _log_int(rng, 1, 14336), width, vocab, dtype, train, rng.choice([0.0, 0.1, 0.3]))
        else:
            case = _distill("", _log_int(rng, 1, 7168), width, vocab, dtype, train, _log_int(rng, 1, 128),
                            rng.choice([1.0, 1.5, 2.0, 4.0]))
    del case["name"]
    return case


# ---- inputs -------------------------------------------------------------------


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _states(g, n, d, table, tokens, dtype):
    """Final states of a trained model: unit-variance rows that lean to their token's embedding, by
    an amount that differs from token to token (confident and unsure positions)."""
    lean = torch.rand((n, 1), generator=g, device="cuda") * 20.0
    return (_normal(g, (n, d)) + lean * (768.0 / d) ** 0.5 * table[tokens].float()).to(dtype)


def _teacher(x, table, k, noise):
    """A teacher's k best logits: those of perturbed states, by blocks of rows."""
    best = [(block @ table.t()).float().topk(k) for block in (x + noise).split(2048)]
    return (torch.cat([b.indices for b in best]).to(torch.int32).contiguous(),
            torch.cat([b.values for b in best]).to(x.dtype).contiguous())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # A residual stream with an offset and a few strong channels, as trained ones have.
        channel = 1.0 + 6.0 * (torch.rand(cols, generator=g, device="cuda") < 0.01).float()
        state["x"] = (_normal(g, (rows, cols)) * channel + 0.25).to(dtype)
        state["residual"] = _normal(g, (rows, cols), 0.5).to(dtype) if case["residual"] else None
        state["gamma"] = 1.0 + _normal(g, (cols,), 0.1)
        state["beta"] = _normal(g, (cols,), 0.1)
        state["dy"] = _normal(g, (rows, cols), 0.1).to(dtype)
        state["dsum"] = _normal(g, (rows, cols), 0.1).to(dtype) if case["residual"] else None
        return state
    n, d, vocab = case["n"], case["d"], case["vocab"]
    table = _normal(g, (vocab, d), 0.02).to(dtype)
    tokens = torch.randint(vocab, (n,), generator=g, device="cuda")
    x = _states(g, n, d, table, tokens, dtype)
    state["x"], state["table"] = x, table
    # Per-token weights of the step: a loss scale over a token count.
    weights = torch.rand(n, generator=g, device="cuda") + 0.5
    state["dloss"] = weights * (64.0 / n ** 0.5)
    if case["op"] == "loss":
        padded = torch.rand(n, generator=g, device="cuda") < case["padding"]
        padded[0] = False
        state["labels"] = torch.where(padded, IGNORE, tokens).to(torch.int32)
    else:
        noise = _normal(g, (n, d), 0.5).to(dtype)
        state["teacher_tokens"], state["teacher_logits"] = _teacher(x, table, min(case["k"], vocab), noise)
    return state


# ---- one pass -----------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "norm":
        return _plain_norm(state)
    if case["op"] == "loss":
        return _plain_loss(case, state)
    return _plain_distill(case, state)


def _run_own(case, s):
    training = importlib.import_module("listenflow-fastest-whisper_b200.training")
    if case["op"] == "norm":
        total, y, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], EPS, residual=s["residual"])
        dx, dgamma, dbeta = training.layer_norm_backward(s["dy"], total, s["gamma"], stats, dsum=s["dsum"])
        out = {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
        if s["residual"] is not None:
            out["sum"] = total
        return out
    if case["op"] == "loss":
        losses, lse = training.cross_entropy_forward(s["x"], s["table"], s["labels"], ignore_index=IGNORE)
        if not case["train"]:
            return {"losses": losses, "lse": lse}
        dx, dtable = training.cross_entropy_backward(s["x"], s["table"], s["labels"], lse, s["dloss"],
                                                     ignore_index=IGNORE)
        return {"losses": losses, "lse": lse, "dx": dx, "dtable": dtable}
    losses, lse = training.distillation_forward(s["x"], s["table"], s["teacher_tokens"], s["teacher_logits"],
                                                temperature=case["temperature"])
    if not case["train"]:
        return {"losses": losses, "lse": lse}
    dx, dtable = training.distillation_backward(s["x"], s["table"], s["teacher_tokens"], s["teacher_logits"], lse,
                                                s["dloss"], temperature=case["temperature"])
    return {"losses": losses, "lse": lse, "dx": dx, "dtable": dtable}


def _plain_norm(s):
    x, dtype = s["x"], s["x"].dtype
    total = x if s["residual"] is None else (x.float() + s["residual"].float()).to(dtype)
    t = total.float()
    centred = t - t.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * s["gamma"] + s["beta"]).to(dtype)
    dy = s["dy"].float()
    dhat = dy * s["gamma"]
    dx = (dhat - dhat.mean(dim=1, keepdim=True) - hat * (dhat * hat).mean(dim=1, keepdim=True)) * rstd
    out = {"y": y, "dgamma": (dy * hat).sum(dim=0), "dbeta": dy.sum(dim=0)}
    if s["residual"] is None:
        out["dx"] = dx.to(dtype)
    else:
        out["dx"] = (dx + s["dsum"].float()).to(dtype)
        out["sum"] = total
    return out


def _softmax_parts(z):
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    return e / total, (top + torch.log(total)).squeeze(1)


def _plain_loss(case, s):
    x, table = s["x"].float(), s["table"].float()
    rows = torch.arange(case["n"], device="cuda")
    valid = s["labels"] != IGNORE
    label = torch.where(valid, s["labels"], 0).long()
    z = x @ table.t()
    p, lse = _softmax_parts(z)
    losses = torch.where(valid, lse - z[rows, label], 0.0)
    if not case["train"]:
        return {"losses": losses, "lse": lse}
    p[rows, label] -= 1.0
    p *= torch.where(valid, s["dloss"], 0.0).unsqueeze(1)
    return {"losses": losses, "lse": lse, "dx": (p @ table).to(s["x"].dtype),
            "dtable": (p.t() @ x).to(s["table"].dtype)}


def _plain_distill(case, s):
    x, table = s["x"].float(), s["table"].float()
    temperature = case["temperature"]
    index = s["teacher_tokens"].long()
    t, t_lse = _softmax_parts(s["teacher_logits"].float() / temperature)
    log_t = s["teacher_logits"].float() / temperature - t_lse.unsqueeze(1)
    z = (x @ table.t()) / temperature
    p, lse = _softmax_parts(z)
    log_p = z.gather(1, index).double() - lse.double().unsqueeze(1)
    losses = (temperature ** 2 * (t * (log_t.double() - log_p)).sum(dim=1)).float()
    if not case["train"]:
        return {"losses": losses, "lse": lse}
    p.scatter_add_(1, index, -t)
    p *= (s["dloss"] * temperature).unsqueeze(1)
    return {"losses": losses, "lse": lse, "dx": (p @ table).to(s["x"].dtype),
            "dtable": (p.t() @ x).to(s["table"].dtype)}


# ---- the definitions in 64 bits ---------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        total = s["x"].double()
        if s["residual"] is not None:  # the sum is held in the rows' type: part of the definition
            total = (total + s["residual"].double()).to(s["x"].dtype).double()
        var, mean = torch.var_mean(total, dim=1, correction=0, keepdim=True)
        rstd = (var + EPS) ** -0.5
        gamma, dy = s["gamma"].double(), s["dy"].double()
        hat = (total - mean) * rstd
        w = dy * gamma
        cols = case["cols"]
        dx = rstd / cols * (cols * w - w.sum(1, keepdim=True) - hat * (w * hat).sum(1, keepdim=True))
        out = {"y": hat * gamma + s["beta"].double(), "dgamma": torch.einsum("rc,rc->c", dy, hat), "dbeta": dy.sum(0)}
        if s["residual"] is None:
            return dict(out, dx=dx)
        return dict(out, dx=dx + s["dsum"].double(), sum=total)
    x, table = s["x"].double(), s["table"].double()
    scale = 1.0 if case["op"] == "loss" else case["temperature"]
    z = (x @ table.T).div_(scale)
    lse = torch.logsumexp(z, dim=1)
    target = torch.zeros_like(z)
    if case["op"] == "loss":
        valid = s["labels"] >= 0
        target[valid.nonzero().squeeze(1), s["labels"][valid].long()] = 1.0
        losses = (lse - (target * z).sum(1)) * valid
    else:
        t = torch.softmax(s["teacher_logits"].double() / scale, dim=1)
        target.scatter_(1, s["teacher_tokens"].long(), t)
        losses = scale ** 2 * (lse + torch.special.xlogy(t, t).sum(1) - (target * z).sum(1))
        valid = torch.ones_like(losses, dtype=torch.bool)
    out = {"losses": losses, "lse": lse}
    if case["train"]:
        dz = z.sub_(lse.unsqueeze(1)).exp_().sub_(target)
        dz *= (s["dloss"].double() * scale * valid).unsqueeze(1)
        out["dx"], out["dtable"] = dz @ table, dz.T @ x
    return out


def work(case):
    if case["op"] == "norm":
        elements = case["rows"] * case["cols"]
        # Forward: x (and residual) in, y (and sum) out; backward: dy, the normalised rows (and dsum) in, dx out.
        moved = 8 if case["residual"] else 5
        return {"bytes": 2 * moved * elements + 16 * case["cols"], "flops": 20 * elements}
    n, d, vocab = case["n"], case["d"], case["vocab"]
    entries = 1 if case["op"] == "loss" else case["k"]
    operands = 2 * d * (n + vocab) + n * (8 + 4 * entries + (2 * entries if case["op"] == "distill" else 0))
    products = 2 * n * vocab * d
    if not case["train"]:
        return {"bytes": operands, "flops": products}
    # The gradients of the states and of the table: one product each, and both tensors written.
    return {"bytes": 2 * operands + 2 * d * (n + vocab), "flops": 3 * products}
