"""Measured cases of the operators on a softmax over a large table (items or words).

  logprobs       log probabilities of given entries, the entropy and the best alternatives of each row
  logprobs_grad  the same with gradients of the log probabilities and the entropy
  distill        a student's loss and gradient against a teacher's best logits
  quantise       rows to microscaled 4-bit floating point (blocks of 32, E2M1 values, E8M0 scales) and back
  product        rows quantised on the way times a table kept in that form: cosine scores, or a layer with a bias

`run` computes them in elementary torch operations in 32 bits; with `own` set it calls recformer_amd.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
INF = float("inf")


# ---- the cases -----------------------------------------------------------------------------------
def listed():
    return [
        # one masked word of one request: a fill-in answer with five alternatives, where latency counts
        {"name": "one masked word", "kind": "logprobs", "m": 1, "n": 50265, "dtype": "bf16", "c": 1, "k": 5,
         "inv_temp": 1.0, "seen": 0},
        # a batch of users against a 10k-item catalog, the items they already have masked, top-50 lists
        {"name": "64 users, 10k items", "kind": "logprobs", "m": 64, "n": 10000, "dtype": "f32", "c": 1, "k": 50,
         "inv_temp": 1.0, "seen": 21},
        # the masked rows of a pretraining batch of 32 sequences: what a teacher answers, 20 best words each
        {"name": "4915 masked rows", "kind": "logprobs", "m": 4915, "n": 50265, "dtype": "bf16", "c": 1, "k": 20,
         "inv_temp": 1.0, "seen": 0},
        # a large catalog with an odd row length (rows of every alignment), four held-out items per user
        {"name": "128 users, 1M items", "kind": "logprobs", "m": 128, "n": 1000003, "dtype": "f32", "c": 4, "k": 50,
         "inv_temp": 0.8, "seen": 50},
        # a training step on log probabilities with an entropy bonus over the masked rows of 16 sequences
        {"name": "2457 rows with gradient", "kind": "logprobs_grad", "m": 2457, "n": 50265, "dtype": "bf16", "c": 1,
         "inv_temp": 1.0},
        # a finetuning batch against a teacher's top-50 items of a 10k catalog
        {"name": "distil 16 users", "kind": "distill", "m": 16, "n": 10000, "dtype": "f32", "k": 50, "temp": 2.0},
        # the masked rows of a pretraining batch against a teacher's 64 best words
        {"name": "distil 4915 rows", "kind": "distill", "m": 4915, "n": 50265, "dtype": "bf16", "k": 64, "temp": 1.0},
        # the queries of one serving batch
        {"name": "quantise 64 queries", "kind": "quantise", "m": 64, "kdim": 768, "dtype": "f16"},
        # a whole catalog, once after every encoding of the items
        {"name": "quantise 1M items", "kind": "quantise", "m": 1000000, "kdim": 768, "dtype": "bf16"},
        # one user against a 1M-item catalog: the table is read once for one row
        {"name": "1 query x 1M items", "kind": "product", "m": 1, "n": 1000000, "kdim": 768, "dtype": "bf16",
         "form": "cos"},
        # an evaluation batch against one of eight shards of a 1M catalog
        {"name": "4096 queries x 125k items", "kind": "product", "m": 4096, "n": 125000, "kdim": 768, "dtype": "f16",
         "form": "cos"},
        # the word decoder of the masked rows of a pretraining batch
        {"name": "decoder of 4915 rows", "kind": "product", "m": 4915, "n": 50265, "kdim": 768, "dtype": "bf16",
         "form": "bias"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "logprobs_grad", "distill", "distill", "quantise", "product", "product"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if kind == "quantise":
        kdim = _log_int(rng, 32, 4096)
        return {"kind": kind, "m": _log_int(rng, 1, min(1000000, 500000000 // kdim)), "kdim": kdim, "dtype": dtype}
    if kind == "product":
        m, kdim = _log_int(rng, 1, 8192), _log_int(rng, 32, 4096)
        n = _log_int(rng, 500, max(501, min(1000000, 300000000000 // (m * kdim), 400000000 // m, 600000000 // kdim)))
        return {"kind": kind, "m": m, "n": n, "kdim": kdim, "dtype": dtype, "form": rng.choice(["cos", "bias"])}
    n = _log_int(rng, 500, 1000000)
    m = _log_int(rng, 1, max(2, min(8192, (120000000 if dtype == "f32" else 240000000) // n)))
    case = {"kind": kind, "m": m, "n": n, "dtype": dtype}
    if kind == "distill":
        return dict(case, k=_log_int(rng, 1, 256), temp=round(rng.uniform(0.5, 4.0), 2))
    case.update(c=_log_int(rng, 1, 8), inv_temp=round(rng.uniform(0.5, 1.5), 2))
    if kind == "logprobs":
        case.update(k=rng.choice([0, 1, _log_int(rng, 2, 256)]), seen=rng.choice([0, 30]))
    return case


def work(case):
    e = SIZE[case["dtype"]]
    m, kind = case["m"], case["kind"]
    if kind == "quantise":  # read the rows, write the codes and scales, read those, write the values
        k = case["kdim"]
        packed = -(-k // 32) * 17
        return {"bytes": m * (2 * k * e + 2 * packed), "flops": 4 * m * k}
    if kind == "product":
        n, k = case["n"], case["kdim"]
        packed = -(-k // 32) * 17
        out = 4 if case["form"] == "cos" else e
        return {"bytes": m * k * e + n * packed + 4 * n + m * n * out, "flops": 2 * m * n * k}
    n = case["n"]
    if kind == "logprobs":
        return {"bytes": m * n * e + m * (12 * case["c"] + 4 + 12 * case["k"]), "flops": 5 * m * n}
    if kind == "logprobs_grad":  # forward reads, backward reads and writes
        return {"bytes": 3 * m * n * e + m * (16 * case["c"] + 8), "flops": 10 * m * n}
    return {"bytes": 3 * m * n * e + 24 * m * case["k"], "flops": 8 * m * n}


# ---- inputs --------------------------------------------------------------------------------------
def _logits(case, gen, dev):
    """Rows as a padded product leaves them: a view with 16-byte aligned rows, one clear answer in most rows."""
    m, n, dt = case["m"], case["n"], DT[case["dtype"]]
    full = torch.empty(m, -(-n // 8) * 8, dtype=dt, device=dev)
    x = full[:, :n]
    x.copy_(torch.randn(m, n, device=dev, generator=gen).mul_(2.0))
    target = torch.randint(0, n, (m,), device=dev, generator=gen)
    rows = torch.arange(m, device=dev)
    x[rows, target] = (6.0 + 4.0 * torch.randn(m, device=dev, generator=gen)).to(dt)
    return x, target, rows


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, m, kind = DT[case["dtype"]], case["m"], case["kind"]
    s = {"case": case}
    if kind in ("logprobs", "logprobs_grad"):
        x, target, rows = _logits(case, gen, dev)
        tokens = torch.randint(0, case["n"], (m, case["c"]), device=dev, generator=gen)
        tokens[:, 0] = target
        if case.get("seen"):  # a user's own history is masked out of the catalog
            seen = torch.randint(0, case["n"], (m, case["seen"]), device=dev, generator=gen)
            keep = x.gather(1, tokens)
            x.scatter_(1, seen, -INF)
            x.scatter_(1, tokens, keep)
        tokens = torch.where(torch.rand(m, case["c"], device=dev, generator=gen) < 0.03,
                             torch.full_like(tokens, -100), tokens)
        tokens[0, 0] = target[0]
        s.update(x=x, tokens=tokens)
        if kind == "logprobs_grad":
            s["g_logp"] = torch.randn(m, case["c"], device=dev, generator=gen) / m
            s["g_entropy"] = torch.full((m,), 0.01 / m, device=dev)
    elif kind == "distill":
        x, _, rows = _logits(case, gen, dev)
        teacher = x.float() * 1.1 + torch.randn(m, case["n"], device=dev, generator=gen)
        values, ids = torch.topk(teacher, min(case["k"], case["n"]), dim=1)
        short = torch.randint(1, case["k"] + 1, (m,), device=dev, generator=gen)  # some lists end early
        short = torch.where(torch.rand(m, device=dev, generator=gen) < 0.1, short, torch.full_like(short, case["k"]))
        slot = torch.arange(ids.shape[1], device=dev)
        s.update(x=x, t_logits=values.contiguous(), t_ids=torch.where(slot < short[:, None], ids, -1))
    else:
        k = case["kdim"]
        spread = torch.rand(k, device=dev, generator=gen) * 1.5 + 0.25  # channels of different size
        s["x"] = (torch.randn(m, k, device=dev, generator=gen) * spread).to(dt)
        if kind == "product":
            n = case["n"]
            table = torch.randn(n, k, device=dev, generator=gen) * (0.05 * spread)
            codes, scales = _quantise(table)
            s["codes"] = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()
            s["scales"] = scales
            if case["form"] == "cos":
                s["rnorm"] = 1.0 / table.square().sum(1).sqrt().clamp_min(1e-8)
            else:
                s["bias"] = torch.randn(n, device=dev, generator=gen)
    return s


# ---- the plain forms -----------------------------------------------------------------------------
def _softmax(x, inv_temp):
    """(z, log of the sum): z = (x - max) * inv_temp in fp32."""
    x = x.float()
    z = (x - x.amax(1, keepdim=True)) * inv_temp
    return z, z.exp().sum(1, keepdim=True).log()


def _entropy(z, lse):
    logp = z - lse
    return -(logp.exp() * logp.clamp_min(-1e30)).sum(1)


def _given(logp, tokens):
    return torch.where(tokens >= 0, logp.gather(1, tokens.clamp_min(0)), torch.zeros((), device=logp.device))


def _logprobs(s):
    case, x, tokens = s["case"], s["x"], s["tokens"]
    z, lse = _softmax(x, case["inv_temp"])
    logp = z - lse
    got = [_given(logp, tokens), _entropy(z, lse)]
    if case["k"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["k"]]
        got += [logp.gather(1, ids), ids]
    return got


def _logprobs_grad(s):
    case, x, tokens = s["case"], s["x"], s["tokens"]
    z, lse = _softmax(x, case["inv_temp"])
    entropy = _entropy(z, lse)
    logp = z - lse
    p = logp.exp()
    g = torch.where(tokens >= 0, s["g_logp"], torch.zeros((), device=x.device))
    d = -p * (g.sum(1, keepdim=True) + s["g_entropy"][:, None] * (logp + entropy[:, None]))
    d.scatter_add_(1, tokens.clamp_min(0), g)
    return [_given(logp, tokens), entropy, (d * case["inv_temp"]).to(x.dtype)]


def _distill(s):
    case, x, ids = s["case"], s["x"], s["t_ids"]
    it = 1.0 / case["temp"]
    z, lse = _softmax(x, it)
    logp = z - lse
    used = ids >= 0
    tz, tlse = _softmax(torch.where(used, s["t_logits"], -INF), it)
    q = (tz - tlse).exp()
    at = ids.clamp_min(0)
    rows = torch.where(used, q * ((tz - tlse).clamp_min(-1e30) - logp.gather(1, at)), 0.0).sum(1)
    d = logp.exp()
    d.scatter_add_(1, at, -q)
    scale = case["temp"] ** 2 / x.shape[0]
    return [rows.sum() * scale, (d * (it * scale)).to(x.dtype)]


def _quantise(x):
    """(codes, scales) of the rows: E2M1 codes, one a byte, of whole blocks, and E8M0 scale bytes."""
    m, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(m, -1, 32)
    top = v.abs().amax(2)
    scale = (torch.frexp(top).exponent + 124).clamp(0, 254)  # 2^(floor(log2 top) - 2), biased by 127
    scale = torch.where(top > 0, scale, torch.zeros_like(scale))
    inv = ((254 - scale) << 23).to(torch.int32).view(torch.float32)
    a = v.abs() * inv[:, :, None]
    code = torch.zeros(a.shape, dtype=torch.uint8, device=x.device)
    code += a > 0.25  # ties go to the even code
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5.0
    code |= (v < 0).to(torch.uint8) << 3
    return code.view(m, -1), scale.to(torch.uint8)


def _values(code, scales, k):
    """fp32 values of codes (one a byte) and scale bytes."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    m = code.shape[0]
    step = (scales.to(torch.int32) << 23).view(torch.float32)  # no scale of these tables is below 1
    return (grid[code.int()].view(m, -1, 32) * step[:, :, None]).reshape(m, -1)[:, :k]


def _product(s):
    case, x = s["case"], s["x"]
    k = case["kdim"]
    a = _values(*_quantise(x), k)
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).flatten(1)
    c = a @ _values(codes, s["scales"], k).t()
    if case["form"] == "cos":
        rn = 1.0 / x.float().square().sum(1).sqrt().clamp_min(1e-8)
        return c * (rn[:, None] * 20.0) * s["rnorm"]
    return (c + s["bias"]).to(x.dtype)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "quantise":
            return _values(*_quantise(state["x"]), case["kdim"]).to(state["x"].dtype)
        return {"logprobs": _logprobs, "logprobs_grad": _logprobs_grad, "distill": _distill, "product": _product}[kind](
            state)
    from recformer_amd import Mxfp4Catalog, ops, train
    x = state["x"]
    if kind == "logprobs":
        r = ops.token_logprobs(x, state["tokens"], k=case["k"], inv_temp=case["inv_temp"], want_entropy=True)
        return [r.logp, r.entropy] + ([r.top_logp, r.top_ids] if case["k"] else [])
    if kind == "logprobs_grad":
        leaf = x.detach().requires_grad_()
        logp, entropy = train.token_logprobs_train(leaf, state["tokens"], inv_temp=case["inv_temp"])
        d, = torch.autograd.grad((logp, entropy), leaf, (state["g_logp"], state["g_entropy"]))
        return [logp.detach(), entropy.detach(), d]
    if kind == "distill":
        leaf = x.detach().requires_grad_()
        loss = train.topk_distill_train(leaf, state["t_logits"], state["t_ids"], temp=case["temp"])
        d, = torch.autograd.grad(loss, leaf)
        return [loss.detach(), d]
    if kind == "quantise":
        return ops.mxfp4_dequantize(ops.mxfp4_quantize(x), x.dtype)
    table = ops.Mxfp4(state["codes"], state["scales"], case["kdim"])
    if case["form"] == "cos":
        return Mxfp4Catalog(table, state["rnorm"]).scores(x, temp=0.05)
    return ops.mxfp4_gemm(x, table, state["bias"], out_dtype=x.dtype)


# ---- in 64 bits ----------------------------------------------------------------------------------
def _grid64(x):
    """The values that rows of x have in 4-bit blocks, in 64 bits: nearest of the grid, the even one of two."""
    m, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(m, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(top.clamp_min(1e-300)))
    e = torch.where(torch.pow(2.0, e + 1) <= top, e + 1, torch.where(torch.pow(2.0, e) > top, e - 1, e))
    step = torch.pow(2.0, (e - 2).clamp(-127, 127))
    a = v / step
    # spacing 1/2 below 2, 1 below 4, 2 above; torch.round takes the even multiple, which is the even code
    gap = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return ((torch.round(a / gap) * gap).clamp(-6, 6) * step).view(m, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    x, kind = s["x"], case["kind"]
    if kind == "quantise":
        return _grid64(x)
    if kind == "product":
        k = case["kdim"]
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        grid = torch.cat([grid, -grid])
        w = torch.stack([grid[(s["codes"] % 16).long()], grid[(s["codes"] // 16).long()]], 2).view(case["n"], -1, 32)
        w = (w * torch.pow(2.0, s["scales"].double() - 127)[:, :, None]).view(case["n"], -1)[:, :k]
        c = _grid64(x) @ w.t()
        if case["form"] == "cos":
            norm = torch.linalg.vector_norm(x.double(), dim=1).clamp_min(1e-8)
            return c.mul_(20.0).div_(norm[:, None]).mul_(s["rnorm"].double())
        return c.add_(s["bias"].double())
    if kind == "distill":
        t = case["temp"]
        ls = torch.log_softmax(x.double() / t, 1)
        lq = torch.log_softmax(s["t_logits"].double().masked_fill(s["t_ids"] < 0, -INF) / t, 1)
        q = lq.exp()
        at = s["t_ids"].clamp_min(0)
        loss = (torch.xlogy(q, q) - q * ls.gather(1, at)).sum() * t * t / case["m"]
        return [loss, (ls.exp().scatter_add(1, at, -q)) * (t / case["m"])]
    it = case["inv_temp"]
    ls = torch.log_softmax(x.double() * it, 1)
    p = ls.exp()
    tokens = s["tokens"]
    logp = ls.gather(1, tokens.clamp_min(0)).masked_fill(tokens < 0, 0.0)
    h = -torch.xlogy(p, p).sum(1)
    if kind == "logprobs":
        if not case["k"]:
            return [logp, h]
        return [logp, h, torch.topk(ls, case["k"], dim=1).values, None]
    g = s["g_logp"].double().masked_fill(tokens < 0, 0.0)
    one = torch.zeros_like(p).scatter_add_(1, tokens.clamp_min(0), g)
    bonus = s["g_entropy"].double()[:, None] * (torch.xlogy(p, p) + p * h[:, None])
    return [logp, h, it * (one - p * g.sum(1, keepdim=True) - bonus)]
