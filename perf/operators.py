"""Cases that time and check the operators on logits and on lists of gradients.

  categorical_logits.adjust / adjust_grad            repetition, presence and frequency penalties, bias, temperature, mask
  categorical_logits.logpdf / sum_logpdf_grad        log-density of a categorical given by logits, value and gradient
  gradients.global_norm / clip_global_norm           2-norm over a list of tensors, and clipping by it

`run` computes them in elementary torch operations, or, where `own` is true, through the framework's entry points."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request's next token: a small vocabulary, a short history, every penalty
        dict(name="adjust-one-row", op="adjust", rows=1, k=32768, dtype="bf16", history=300, penalties=True, bias="none",
             mask="none", temperature=True),
        # a decode step of a server: 64 requests, long ragged histories, a grammar's packed mask per request
        dict(name="adjust-decode-batch", op="adjust", rows=64, k=131072, dtype="bf16", history=2048, penalties=True,
             bias="none", mask="bits", temperature=True),
        # a large batch in float32 over an odd number of categories, a bias shared by all rows
        dict(name="adjust-odd-f32", op="adjust", rows=256, k=100003, dtype="f32", history=4001, penalties=True,
             bias="shared", mask="none", temperature=True),
        # training under a constraint: boolean mask per row, learned shared bias, gradients of both
        dict(name="adjust-grad-train", op="adjust_grad", rows=4096, k=32768, dtype="bf16", history=0, penalties=False,
             bias="shared", mask="bool", temperature=True),
        # scoring one token per request
        dict(name="logpdf-decode", op="logpdf", rows=8, k=50021, dtype="f32"),
        # scoring a whole corpus batch
        dict(name="logpdf-score", op="logpdf", rows=8192, k=32768, dtype="f16"),
        # a classifier's step: few categories, float64
        dict(name="logpdf-grad-small-f64", op="logpdf_grad", rows=256, k=1000, dtype="f64"),
        # odd number of categories in float32
        dict(name="logpdf-grad-odd-f32", op="logpdf_grad", rows=1500, k=100003, dtype="f32"),
        # a training step of a model with many categories
        dict(name="logpdf-grad-train", op="logpdf_grad", rows=4096, k=131072, dtype="bf16"),
        # the norm of a small model's gradients, for a log line
        dict(name="norm-small", op="norm", tensors=24, total=60000, dtype="f32", odd=True),
        # clipping the gradients of a large model
        dict(name="clip-large", op="clip", tensors=290, total=640000000, dtype="bf16", odd=False, clips=True),
        # clipping float32 gradients of odd sizes
        dict(name="clip-odd-f32", op="clip", tensors=61, total=40000000, dtype="f32", odd=True, clips=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("adjust", "adjust", "adjust_grad", "logpdf", "logpdf_grad", "norm", "clip"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32", "f32", "f64"))
    if op in ("norm", "clip"):
        tensors = _log_uniform(rng, 1, 320)
        total = max(tensors, _log_uniform(rng, 2000, 100000000))
        case = dict(op=op, tensors=tensors, total=total, dtype=dtype, odd=rng.random() < 0.5)
        if op == "clip":
            case["clips"] = rng.random() < 0.8
        return case
    k = _log_uniform(rng, 1000, 160000)
    rows = _log_uniform(rng, 1, max(2, min(8192, 400000000 // DTYPES[dtype].itemsize // k)))
    case = dict(op=op, rows=rows, k=k, dtype=dtype)
    if op.startswith("adjust"):
        penalties = rng.random() < (0.75 if op == "adjust" else 0.4)
        case.update(history=_log_uniform(rng, 1, 8000 if rows <= 1024 else 500) if penalties else 0, penalties=penalties,
                    bias=rng.choice(("none", "shared", "rows")), mask=rng.choice(("none", "bool", "bits")),
                    temperature=rng.random() < 0.7)
    return case


# ---------------------------------------------------------------------------------------------- prepare
def _sizes(case):
    """Sizes of a list of tensors: most of the elements in matrices, every third one a short vector."""
    n, total = case["tensors"], case["total"]
    weights = [1.0 / 500 if i % 3 == 2 else 1.0 + (i * 7 % 5) / 4 for i in range(n)]
    sizes = [max(1, int(total * w / sum(weights))) for w in weights]
    return [s | 1 for s in sizes] if case["odd"] else [max(1, s - s % 64) for s in sizes]


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    state = {"case": case}
    if case["op"] in ("norm", "clip"):
        sizes = _sizes(case)
        grads = [(torch.randn(n, generator=gen, device=device, dtype=torch.float32) * 0.02).to(dtype) for n in sizes]
        state["grads"] = grads
        if case["op"] == "clip":
            norm = 0.02 * math.sqrt(sum(sizes))
            state["max_norm"] = 0.3 * norm if case["clips"] else 3.0 * norm
            places = [0]
            for n in sizes:  # every output starts on a 256-byte border of one buffer
                places.append(places[-1] + (n + 127) // 128 * 128)
            state["flat"] = torch.zeros(places[-1], dtype=dtype, device=device)
            state["out"] = [state["flat"][p : p + n] for p, n in zip(places, sizes)]
        return state
    rows, k = case["rows"], case["k"]
    state["logits"] = (torch.randn(rows, k, generator=gen, device=device, dtype=torch.float32) * 2.5).to(dtype)
    if case["op"].startswith("logpdf"):
        x = torch.randint(0, k, (rows,), generator=gen, device=device)
        state["x"] = x
        if case["op"] == "logpdf_grad":  # one row in eight is padding
            pad = torch.rand(rows, generator=gen, device=device) < 0.125
            state["x"] = torch.where(pad, -1, x)
            state["weights"] = torch.where(pad, 0.0, 1.0).to(wide)
        return state
    args = {}

    def per_row(lo, hi):
        return lo + (hi - lo) * torch.rand(rows, generator=gen, device=device, dtype=wide)

    if case["penalties"]:
        n = case["history"]
        # text repeats itself: ids piled up near zero, as in a vocabulary ordered by frequency
        u = torch.rand(rows, n, generator=gen, device=device)
        args["history"] = ((k - 1) * u * u * u).to(torch.int64)
        args["lengths"] = torch.randint(0, n + 1, (rows,), generator=gen, device=device)
        args["prompt_lengths"] = torch.randint(0, n + 1, (rows,), generator=gen, device=device) // 2
        args["repetition"] = per_row(1.0, 1.4)
        args["presence"] = per_row(0.0, 0.8)
        args["frequency"] = per_row(0.0, 0.3)
    if case["temperature"]:
        args["temperature"] = per_row(0.6, 1.2)
    if case["bias"] != "none":
        args["bias"] = torch.randn(*(() if case["bias"] == "shared" else (rows,)), k, generator=gen, device=device, dtype=wide)
    if case["mask"] != "none":
        share = torch.rand(rows, 1, generator=gen, device=device)  # a grammar allows few categories here, most there
        allowed = torch.rand(rows, k, generator=gen, device=device) < share
        args["mask"] = allowed if case["mask"] == "bool" else _packed(allowed)
    state["args"] = args
    if case["op"] == "adjust_grad":
        state["g"] = (torch.randn(rows, k, generator=gen, device=device, dtype=torch.float32) * 0.1).to(dtype)
    return state


def _packed(allowed):
    """(rows, k) truth values as (rows, ceil(k / 32)) words: category v is bit v % 32 of word v // 32."""
    rows, k = allowed.shape
    words = (k + 31) // 32
    bits = torch.zeros(rows, words * 32, dtype=torch.int64, device=allowed.device)
    bits[:, :k] = allowed
    w = (bits.reshape(rows, words, 32) << torch.arange(32, device=allowed.device)).sum(dim=2)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


# -------------------------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        from distributions_amd import categorical_logits, gradients

        if op == "adjust":
            return categorical_logits.adjust(state["logits"], **state["args"])
        if op == "adjust_grad":
            g_logits, g_bias = categorical_logits.adjust_grad(state["g"], state["logits"], **state["args"])
            return [g_logits] if g_bias is None else [g_logits, g_bias]
        if op == "logpdf":
            return categorical_logits.logpdf(state["x"], state["logits"])
        if op == "logpdf_grad":
            total, grads = categorical_logits.sum_logpdf_grad(state["x"], state["logits"], state["weights"])
            return [total, grads[1]]
        if op == "norm":
            return gradients.global_norm(state["grads"])
        norm, _ = gradients.clip_global_norm(state["grads"], state["max_norm"], out=state["out"])
        return [norm, state["flat"]]
    if op == "adjust":
        return _adjust(state["logits"], **state["args"])
    if op == "adjust_grad":
        return _adjust_grad(state["g"], state["logits"], **state["args"])
    if op == "logpdf":
        return _logpdf(state["x"], state["logits"])[0]
    if op == "logpdf_grad":
        return _logpdf_grad(state["x"], state["logits"], state["weights"])
    if op == "norm":
        return _norm(state["grads"])
    return _clip(state["grads"], state["max_norm"], state["out"], state["flat"])


def _wide(t):
    return t if t.dtype == torch.float64 else t.to(torch.float32)


def _counts(history, first, last, k):
    """How often each category stands in history[r, first[r]:last[r]]."""
    at = torch.arange(history.shape[1], device=history.device)
    within = (at >= first[:, None]) & (at < last[:, None]) & (history >= 0) & (history < k)
    counts = torch.zeros(history.shape[0], k + 1, dtype=torch.int32, device=history.device)
    counts.scatter_add_(1, torch.where(within, history, k), torch.ones_like(history, dtype=torch.int32))
    return counts[:, :k]


def _allowed(mask, k):
    if mask.dtype == torch.bool:
        return mask
    v = torch.arange(k, device=mask.device)
    return (mask[:, v // 32] >> (v % 32).to(torch.int32)) & 1 == 1


def _adjust(logits, history=None, lengths=None, prompt_lengths=None, repetition=None, presence=None, frequency=None,
            bias=None, temperature=None, mask=None):
    x = _wide(logits)
    k = x.shape[1]
    if history is not None:
        seen = _counts(history, torch.zeros_like(lengths), lengths, k) > 0
        made = _counts(history, prompt_lengths, lengths, k)
        rho = repetition[:, None]
        x = torch.where(seen, torch.where(x > 0, x / rho, x * rho), x)
        x = x - (frequency[:, None] * made + presence[:, None] * (made > 0))
    if bias is not None:
        x = x + bias
    if temperature is not None:
        x = x / temperature[:, None]
    if mask is not None:
        x = torch.where(_allowed(mask, k), x, -math.inf)
    return x.to(logits.dtype)


def _adjust_grad(g, logits, history=None, lengths=None, prompt_lengths=None, repetition=None, presence=None,
                 frequency=None, bias=None, temperature=None, mask=None):
    d = _wide(g)
    k = d.shape[1]
    if mask is not None:
        d = torch.where(_allowed(mask, k), d, 0.0)
    if temperature is not None:
        d = d / temperature[:, None]
    g_bias = None
    if bias is not None:
        g_bias = d.sum(dim=0) if bias.dim() == 1 else d.to(bias.dtype)
    if history is not None:
        seen = _counts(history, torch.zeros_like(lengths), lengths, k) > 0
        rho = repetition[:, None]
        d = torch.where(seen, torch.where(logits > 0, d / rho, d * rho), d)
    d = d.to(logits.dtype)
    return [d] if g_bias is None else [d, g_bias]


def _logpdf(x, logits):
    z = _wide(logits)
    m = z.max(dim=1, keepdim=True).values
    e = (z - m).exp()
    s = e.sum(dim=1, keepdim=True)
    inside = (x >= 0) & (x < z.shape[1])
    zx = z.gather(1, torch.where(inside, x, 0)[:, None])
    return torch.where(inside, (zx - m - s.log())[:, 0], -math.inf), e, s, inside


def _logpdf_grad(x, logits, weights):
    lp, e, s, inside = _logpdf(x, logits)
    total = torch.where(weights == 0, 0.0, weights * lp).double().sum().to(lp.dtype)
    w = torch.where(inside, weights, 0.0)[:, None]
    d = e * (-w / s)
    d.scatter_add_(1, torch.where(inside, x, 0)[:, None], w)
    return [total, d.to(logits.dtype)]


def _norm(grads):
    return torch.stack([_wide(g).square().sum() for g in grads]).double().sum().sqrt().to(_wide(grads[0]).dtype)


def _clip(grads, max_norm, out, flat):
    norm = _norm(grads)
    scale = torch.where(norm > max_norm, max_norm / norm, 1.0)
    _ = [o.copy_(_wide(g) * scale) for g, o in zip(grads, out)]
    return [norm, flat]


# ------------------------------------------------------------------------------------------------- work
def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] in ("norm", "clip"):
        n = sum(_sizes(case))
        return {"bytes": n * size * (2 if case["op"] == "clip" else 1), "flops": n * (3 if case["op"] == "clip" else 2)}
    rows, k = case["rows"], case["k"]
    n = rows * k
    if case["op"] == "logpdf":
        return {"bytes": n * size + 12 * rows, "flops": 4 * n}
    if case["op"] == "logpdf_grad":
        return {"bytes": 2 * n * size + 12 * rows, "flops": 8 * n}
    wide = 8 if case["dtype"] == "f64" else 4
    total = 2 * n * size + {"none": 0, "bool": n, "bits": 4 * rows * ((k + 31) // 32)}[case["mask"]]
    total += {"none": 0, "shared": k * wide, "rows": n * wide}[case["bias"]]
    if case["penalties"]:  # half of a ragged history on average
        total += rows * (4 * case["history"] + 16 + 3 * wide)
    return {"bytes": total + (rows * wide if case["temperature"] else 0), "flops": 4 * n}


# ------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """The definitions in 64 bits, row block by row block."""
    state = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op in ("norm", "clip"):
        squares = [float(torch.dot(c, c)) for g in state["grads"] for c in g.to(f64).split(1 << 24)]
        norm = math.sqrt(math.fsum(squares))
        if op == "norm":
            return torch.tensor(norm, dtype=f64)
        flat = state["flat"].to(f64)
        factor = state["max_norm"] / norm if norm > state["max_norm"] else 1.0
        start = 0
        for g in state["grads"]:
            flat[start : start + g.numel()] = g.to(f64).mul_(factor)
            start += (g.numel() + 127) // 128 * 128
        return [torch.tensor(norm, dtype=f64), flat]
    logits = state["logits"]
    rows, k = logits.shape
    step = max(1, (1 << 27) // k)
    blocks = [slice(r, min(rows, r + step)) for r in range(0, rows, step)]
    if op.startswith("logpdf"):
        lps, grads, total = [], [], 0.0
        for b in blocks:
            logp = logits[b].to(f64).log_softmax(dim=1)
            x = state["x"][b]
            ok = (x >= 0) & (x < k)
            lp = logp[torch.arange(len(x), device=x.device), x.clamp(0, k - 1)]
            lps.append(torch.where(ok, lp, torch.full_like(lp, -math.inf)))
            if op == "logpdf_grad":
                w = state["weights"][b].to(f64)
                keep = w != 0
                total += float((w[keep] * lps[-1][keep]).sum())
                hot = torch.zeros_like(logp)
                hot[torch.arange(len(x), device=x.device), x.clamp(0, k - 1)] = 1.0
                grads.append((hot - logp.exp()) * (w * ok)[:, None])
        if op == "logpdf":
            return torch.cat(lps)
        return [torch.tensor(total, dtype=f64), torch.cat(grads)]
    a = state["args"]
    outs, shared, per_row = [], torch.zeros(k, dtype=f64, device=logits.device), []
    for b in blocks:
        z = logits[b].to(f64)
        n = z.shape[0]
        t = a["temperature"][b].to(f64).view(n, 1) if "temperature" in a else torch.ones(n, 1, dtype=f64, device=z.device)
        if "mask" in a:
            m = a["mask"][b]
            if m.dtype != torch.bool:
                words = (m.to(torch.int64) & 0xFFFFFFFF).unsqueeze(2)
                m = ((words // (2 ** torch.arange(32, device=m.device))) % 2 == 1).reshape(n, -1)[:, :k]
        else:
            m = torch.ones_like(z, dtype=torch.bool)
        factor = torch.ones_like(z)
        minus = torch.zeros_like(z)
        if "history" in a:
            h = a["history"][b]
            place = torch.arange(h.shape[1], device=h.device).expand_as(h)
            row = torch.arange(n, device=h.device).view(n, 1).expand_as(h)
            upto = place < a["lengths"][b].view(n, 1)
            since = upto & (place >= a["prompt_lengths"][b].view(n, 1))
            rho = a["repetition"][b].to(f64).view(n, 1)
            seen = torch.bincount((row * k + h)[upto], minlength=n * k).reshape(n, k)
            factor = torch.where(seen > 0, torch.where(z > 0, 1.0 / rho, rho), factor)
            made = torch.bincount((row * k + h)[since], minlength=n * k).reshape(n, k).to(f64)
            minus = made * a["frequency"][b].to(f64).view(n, 1) + made.clamp(max=1) * a["presence"][b].to(f64).view(n, 1)
        if op == "adjust":
            s = z * factor - minus
            if "bias" in a:
                s = s + (a["bias"] if a["bias"].dim() == 1 else a["bias"][b]).to(f64)
            outs.append((s / t).masked_fill(~m, -math.inf))
            continue
        d = state["g"][b].to(f64) * m / t
        if "bias" in a:
            if a["bias"].dim() == 1:
                shared += d.sum(dim=0)
            else:
                per_row.append(d)
        outs.append(d * factor)
    if op == "adjust":
        return torch.cat(outs)
    if "bias" not in a:
        return [torch.cat(outs)]
    return [torch.cat(outs), shared if a["bias"].dim() == 1 else torch.cat(per_row)]
