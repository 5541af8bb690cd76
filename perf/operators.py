"""Performance cases of the score operators: what a program calls that trains an embedding
model against neighbour lists or another model's scores, and answers queries from its table.

Kinds (one pass each):
  product   scores of M rows against a table of N rows, both in 8 bits with a scale for each
            block of 128 ("b": the table's scales by row or by 128 x 128 square)
  grad      gradients of such a product: its upstream gradient brought to 8 bits, then the
            products with the transposed table and the transposed input
  quantize  rows to 8 bits ("block": row or square scales), with the transposed copy or without
  top       the first k scores of each row in (score, id) order and the row's log-sum-exp
  distill   the loss against a teacher's top scores with its gradient: one call, or forward
            and backward apart ("apart"); "tail" = the teacher's log-sum-exp is known and its
            remaining mass counts against the student's

Scores ("type": bf16, fp16 or fp32) have rows "pad" elements apart beyond their length;
"masked" is the share of columns at -inf (rows filtered out).
"""
import math

import torch

own = False

BLOCK = 128       # columns a scale stands for
LARGEST = 448.0   # largest finite value of the 8-bit type (e4m3)
SMALLEST = 2.0 ** -64  # a block's largest magnitude counts as this at least
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _product(name, m, n, d, b, out):
    return dict(name=name, kind="product", m=m, n=n, d=d, b=b, out=out)


def _grad(name, m, n, d):
    return dict(name=name, kind="grad", m=m, n=n, d=d)


def _quantize(name, n, d, type, block, transpose):
    return dict(name=name, kind="quantize", n=n, d=d, type=type, block=block, transpose=transpose)


def _top(name, n, v, k, type, temperature=1.0, pad=0, masked=0.0):
    return dict(name=name, kind="top", n=n, v=v, k=k, type=type, temperature=temperature, pad=pad, masked=masked)


def _distill(name, n, v, k, type, tail, apart, temperature=1.0, pad=0, masked=0.0):
    return dict(name=name, kind="distill", n=n, v=v, k=k, type=type, tail=tail, apart=apart, temperature=temperature,
                pad=pad, masked=masked)


def listed():
    return [
        # one query against a small table: launches and waits count
        _product("score_1x10k_d128", 1, 10_000, 128, "row", "fp32"),
        # a ragged batch of queries against a table of text embeddings
        _product("score_77x100k_d384", 77, 100_000, 384, "row", "bf16"),
        # scores of a training batch at embedding width against a vocabulary
        _product("head_4096x32768_d768", 4096, 32_768, 768, "square", "bf16"),
        # a model's square layer: long sums
        _product("layer_4096x4096_d4096", 4096, 4096, 4096, "square", "bf16"),
        # gradients of a small odd batch
        _grad("grad_300x1000_d100", 300, 1000, 100),
        # gradients of the head
        _grad("grad_4096x32768_d768", 4096, 32_768, 768),
        # a whole base set becomes a table
        _quantize("table_1m_d384", 1_000_000, 384, "fp32", "row", False),
        # an odd batch of activations, kept both ways round for the backward pass
        _quantize("rows_4097_d768", 4097, 768, "bf16", "row", True),
        # the best of one query's scores
        _top("top_1x100k_k32", 1, 100_000, 32, "bf16"),
        # a teacher's top scores of a training batch
        _top("top_4096x32768_k64", 4096, 32_768, 64, "bf16", temperature=2.0),
        # a small batch against the exact lists of a small base set, half its rows filtered out
        _distill("distill_64x10000_k32", 64, 10_000, 32, "fp32", False, True, temperature=0.5, masked=0.5),
        # a training batch against another model's top scores
        _distill("distill_4096x32768_k64", 4096, 32_768, 64, "bf16", True, False, temperature=2.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["product", "product", "grad", "quantize", "top", "distill", "distill"])
    d = rng.choice([64, 100, 128, 128, 384, 384, 768, 768, 1024, 2048, 4096, _log_int(rng, 17, 2000)])
    if kind == "product":
        m, n = _log_int(rng, 1, 8192), _log_int(rng, 500, 300_000)
        while m * n * d > 100_000_000_000 or m * n > 130_000_000:
            m, n = (m + 1) // 2, n if m > 64 else n * 2 // 3
        c = _product(None, m, n, d, rng.choice(["row", "square"]), rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    elif kind == "grad":
        m, n = _log_int(rng, 16, 8192), _log_int(rng, 200, 60_000)
        while m * n * d > 100_000_000_000 or m * n > 130_000_000:
            m, n = (m + 1) // 2, n if m > 64 else n * 2 // 3
        c = _grad(None, m, n, d)
    elif kind == "quantize":
        n = _log_int(rng, 1, 300_000)
        while n * d > 200_000_000:
            n = n * 2 // 3
        c = _quantize(None, n, d, rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["row", "row", "square"]),
                      rng.random() < 0.5)
    else:
        type = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        n, v = _log_int(rng, 1, 8192), _log_int(rng, 50, 1_000_000)
        while n * v > (60_000_000 if type == "fp32" else 130_000_000):
            n = (n + 1) // 2
        common = dict(temperature=rng.choice([0.5, 1.0, 2.0]), pad=rng.choice([0, 0, 8, 24, 1, 3]),
                      masked=rng.choice([0.0, 0.0, 0.3, 0.9]))
        if kind == "top":
            c = _top(None, n, v, rng.choice([1, 6, 20, 32, 64, 100, 128]), type, **common)
        else:
            c = _distill(None, n, v, rng.choice([1, 6, 20, 32, 64, 100, 128]), type, rng.random() < 0.5,
                         rng.random() < 0.5, **common)
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------------
def _ceil(n):
    return -(-n // BLOCK)


def _quantized(x, block):
    """(8-bit rows padded to whole blocks, scales) of x in the plain form."""
    n, d = x.shape
    f = torch.nn.functional.pad(x.float(), (0, _ceil(d) * BLOCK - d))
    if block == "row":
        f = f.view(n, 1, _ceil(d), BLOCK)
    else:
        f = torch.nn.functional.pad(f, (0, 0, 0, _ceil(n) * BLOCK - n)).view(_ceil(n), BLOCK, _ceil(d), BLOCK)
    scale = f.abs().amax(dim=(1, 3), keepdim=True).clamp(min=SMALLEST) / LARGEST
    q = (f / scale).to(torch.float8_e4m3fn)
    return q.view(-1, _ceil(d) * BLOCK)[:n].contiguous(), scale[:, 0, :, 0].contiguous()


def _transposed(q, n, d, scale):
    """The same 8-bit values the other way round (square scales turn with them)."""
    t = torch.zeros(d, _ceil(n) * BLOCK, dtype=torch.uint8, device=q.device)
    t[:, :n] = q.view(torch.uint8)[:, :d].t()
    return t.view(torch.float8_e4m3fn), scale.t().contiguous()


def _rows(g, n, d):
    """Embeddings: rows of a Gaussian mixture of 64 centroids at unit length."""
    x = torch.randn(64, d, device="cuda", generator=g)[torch.randint(0, 64, (n,), device="cuda", generator=g)]
    x += 0.6 * torch.randn(n, d, device="cuda", generator=g)
    return x / x.norm(dim=1, keepdim=True)


def _scores(case, g):
    """Scores [n, v] at the case's row distance, some columns of each row filtered out."""
    n, v = case["n"], case["v"]
    whole = torch.empty(n, v + case["pad"], dtype=TYPES[case["type"]], device="cuda")
    step = max(1, (1 << 26) // v)
    for i in range(0, n, step):
        x = torch.randn(min(step, n - i), v, device="cuda", generator=g) * 2.5
        if case["masked"]:
            x.masked_fill_(torch.rand(x.shape, device="cuda", generator=g) < case["masked"], -math.inf)
        whole[i:i + step, :v] = x
    return whole[:, :v]


def _teacher(case, s, g):
    """A teacher's top scores (ids, scores, log-sum-exp over all its scores): near the
    student's own, in descending order, the last ones of some rows missing, and now and then
    a row without any."""
    n, v, k = case["n"], case["v"], case["k"]
    ids = torch.full((n, k), -1, dtype=torch.int32, device="cuda")
    m = min(k, v)
    step = v // m  # distinct ids: one of each of m stretches of the row
    ids[:, :m] = (torch.arange(m, device="cuda") * step
                  + torch.randint(0, step, (n, m), device="cuda", generator=g)).int()
    val = (torch.randn(n, k, device="cuda", generator=g) * 1.5 + 4.0).sort(dim=1, descending=True).values
    lse = torch.logsumexp(val / case["temperature"], dim=1) + 0.05 + torch.rand(n, device="cuda", generator=g)
    keep = torch.randint(k - k // 4, k + 1, (n, 1), device="cuda", generator=g)
    keep[torch.rand(n, 1, device="cuda", generator=g) < 0.02] = 0
    gone = (torch.arange(k, device="cuda") >= keep) | (ids < 0)
    # what the student has filtered out, the teacher's list does not hold either
    gone |= s.gather(1, ids.clamp(min=0).long()) == -math.inf
    return ids.masked_fill(gone, -1), val.masked_fill(gone, -math.inf), lse


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    s = {"case": case}
    kind = case["kind"]
    if kind == "product":
        s["a"], s["a_scale"] = _quantized(_rows(g, case["m"], case["d"]), "row")
        s["b"], s["b_scale"] = _quantized(_rows(g, case["n"], case["d"]), case["b"])
    elif kind == "grad":
        m, n, d = case["m"], case["n"], case["d"]
        x, w = _rows(g, m, d).bfloat16(), _rows(g, n, d).bfloat16()
        up = torch.softmax(torch.randn(m, n, device="cuda", generator=g) * 3, dim=1)
        up[torch.arange(m, device="cuda"), torch.randint(0, n, (m,), device="cuda", generator=g)] -= 1
        s["g"] = (up / m).bfloat16()
        s["xt"], s["xt_scale"] = _quantized(x.t(), "row")  # kept by the forward pass
        q, scale = _quantized(w, "square")
        s["wt"], s["wt_scale"] = _transposed(q, n, d, scale)
    elif kind == "quantize":
        s["x"] = torch.empty(case["n"], case["d"], dtype=TYPES[case["type"]], device="cuda")
        for i in range(0, case["n"], 1 << 17):
            s["x"][i:i + (1 << 17)] = _rows(g, min(1 << 17, case["n"] - i), case["d"])
    else:
        s["scores"] = _scores(case, g)
        if kind == "distill":
            s["ids"], s["values"], s["lse"] = _teacher(case, s["scores"], g)
            if not case["tail"]:
                s["lse"] = None
            s["weight"] = torch.rand(case["n"], device="cuda", generator=g) / case["n"]  # of each row's loss
    return s


# ---- the plain forms ----------------------------------------------------------------
def _values(q, scale):
    """What 8-bit rows stand for, in 32 bits."""
    n, d = q.shape
    if scale.shape[0] != n:
        scale = scale.repeat_interleave(BLOCK, dim=0)[:n]
    return (q.float().view(n, d // BLOCK, BLOCK) * scale[:, :, None]).view(n, d)


def _plain_grad(s):
    g = s["g"]
    m, n = g.shape
    gq, gs = _quantized(g, "row")
    gt, gts = _quantized(g.t(), "row")
    dx = _values(gq, gs) @ _values(s["wt"], s["wt_scale"]).t()
    dw = _values(gt, gts) @ _values(s["xt"], s["xt_scale"]).t()
    return dx.bfloat16(), dw


def _plain_quantize(s, case):
    x = s["x"]
    q, scale = _quantized(x, case["block"])
    if not case["transpose"]:
        return q, scale
    if case["block"] == "row":
        return (q, scale) + _quantized(x.t(), "row")
    return (q, scale) + _transposed(q, *x.shape, scale)


def _lse(x):
    top = x.amax(dim=1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    return top[:, 0] + (x - top).exp().sum(dim=1).log()


def _plain_top(s, case):
    x = s["scores"].float() + 0.0  # -0 counts as 0
    n, v = x.shape
    bits = x.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    order = torch.where(x.isnan(), torch.full_like(order, 0x7FFFFFFF), order)
    keys = (order.long() << 32) | (0xFFFFFFFF - torch.arange(v, device=x.device))
    m = min(case["k"], v)
    ids = torch.full((n, case["k"]), -1, dtype=torch.int32, device=x.device)
    val = torch.full((n, case["k"]), -math.inf, device=x.device)
    at = 0xFFFFFFFF - (keys.topk(m, dim=1).values & 0xFFFFFFFF)
    val[:, :m] = x.gather(1, at)
    ids[:, :m] = torch.where(val[:, :m] == -math.inf, torch.full_like(at, -1), at).int()
    return val, ids, _lse(x / case["temperature"])


def _loss_and_gradient(scores, ids, values, lse, weight, temperature):
    """Loss of each row and the scores' gradient, in the type of `scores`."""
    n, v = scores.shape
    x = scores / temperature
    there = (ids >= 0) & (ids < v) & (values != -math.inf)
    at = torch.where(there, ids, torch.zeros_like(ids)).long()
    t = (values / temperature).masked_fill(~there, -math.inf)
    top = x.amax(dim=1, keepdim=True)
    full = there.any(dim=1, keepdim=True) & (top != -math.inf)
    top = torch.where(full, top, torch.zeros_like(top))
    e = (x - top).exp()
    total = e.sum(dim=1, keepdim=True)
    if lse is None:
        t_top = torch.where(full, t.amax(dim=1, keepdim=True), torch.zeros_like(top))
        log_p = t - t_top - (t - t_top).exp().sum(dim=1, keepdim=True).log()
    else:
        log_p = t - lse[:, None].to(x.dtype)
    p = log_p.exp()
    log_q = x.gather(1, at) - top - total.log()
    loss = torch.where(there & (p > 0), p * (log_p - log_q), torch.zeros_like(p)).sum(dim=1, keepdim=True)
    mass = p.sum(dim=1, keepdim=True)
    q = e / total
    if lse is None:
        grad = mass * q
    else:
        listed_ = torch.zeros_like(e).scatter_add_(1, at, there.to(e.dtype)) > 0
        rest_x = x.masked_fill(listed_, -math.inf)
        rest_top = rest_x.amax(dim=1, keepdim=True)
        some = (rest_top > -math.inf) & (mass < 1)
        rest_top = torch.where(some, rest_top, top)
        rest_e = (rest_x - rest_top).exp()
        rest_total = torch.where(some, rest_e.sum(dim=1, keepdim=True), torch.ones_like(mass))
        rest = torch.where(some, 1 - mass, torch.zeros_like(mass))
        log_rest_q = rest_top + rest_total.log() - top - total.log()
        loss = loss + torch.where(some, rest * (rest.log() - log_rest_q), torch.zeros_like(rest))
        grad = q * (mass + rest) - rest_e * (rest / rest_total)
    grad = grad.scatter_add(1, at, torch.where(there, -p, torch.zeros_like(p)))
    grad = grad * (weight[:, None].to(x.dtype) / temperature)
    return (torch.where(full, loss, torch.zeros_like(loss))[:, 0],
            torch.where(full, grad, torch.zeros_like(grad)))


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from filtervectorcode_refactor_amd import scores
        if kind == "product":
            return scores.matmul_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"], dtype=TYPES[case["out"]])
        if kind == "grad":
            return scores.matmul_fp8_grad(s["g"], s["xt"], s["xt_scale"], s["wt"], s["wt_scale"])
        if kind == "quantize":
            return scores.quantize_fp8(s["x"], block=case["block"], transpose=case["transpose"])
        if kind == "top":
            return scores.top_scores(s["scores"], case["k"], temperature=case["temperature"])
        if not case["apart"]:
            return scores.distill_step(s["scores"], s["ids"], s["values"], s["weight"], teacher_lse=s["lse"],
                                       temperature=case["temperature"])
        loss, saved = scores.distill_forward(s["scores"], s["ids"], s["values"], teacher_lse=s["lse"],
                                             temperature=case["temperature"])
        return loss, scores.distill_backward(s["weight"], s["scores"], s["ids"], s["values"], saved,
                                             teacher_lse=s["lse"], temperature=case["temperature"])
    if kind == "product":
        return (_values(s["a"], s["a_scale"]) @ _values(s["b"], s["b_scale"]).t()).to(TYPES[case["out"]])
    if kind == "grad":
        return _plain_grad(s)
    if kind == "quantize":
        return _plain_quantize(s, case)
    if kind == "top":
        return _plain_top(s, case)
    loss, grad = _loss_and_gradient(s["scores"].float(), s["ids"], s["values"], s["lse"], s["weight"],
                                    case["temperature"])
    return loss, grad.to(TYPES[case["type"]])


# ---- what a pass cannot do without --------------------------------------------------
def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind == "product":
        m, n, d = case["m"], case["n"], case["d"]
        scales = 4 * _ceil(d) * (m + (n if case["b"] == "row" else _ceil(n)))
        return {"bytes": (m + n) * d + scales + m * n * size[case["out"]], "flops": 2 * m * n * d}
    if kind == "grad":
        m, n, d = case["m"], case["n"], case["d"]
        return {"bytes": 2 * m * n + (m + n) * d + 2 * m * d + 4 * n * d, "flops": 4 * m * n * d}
    if kind == "quantize":
        n, d = case["n"], case["d"]
        copies = 2 if case["transpose"] else 1
        return {"bytes": n * d * size[case["type"]] + copies * n * d, "flops": 3 * copies * n * d}
    n, v, k = case["n"], case["v"], case["k"]
    if kind == "top":
        return {"bytes": n * v * size[case["type"]] + n * (8 * k + 4), "flops": 4 * n * v}
    return {"bytes": 2 * n * v * size[case["type"]] + n * (8 * k + 12), "flops": 8 * n * v}


# ---- the definitions in 64 bits -----------------------------------------------------
def _expand(q, scale):
    """8-bit rows and their scales as 64-bit values."""
    rows = torch.arange(q.shape[0], device=q.device)
    cols = torch.arange(q.shape[1], device=q.device) // BLOCK
    if scale.shape[0] != q.shape[0]:
        rows = rows // BLOCK
    return q.to(torch.float64) * scale.double()[rows][:, cols]


def _exact_scales(x, block):
    """(values / scale as the 8-bit type holds them, scales): the scale is the 32-bit one, it
    is part of the definition."""
    n, d = x.shape
    out = torch.zeros(n, _ceil(d) * BLOCK, dtype=torch.float64, device=x.device)
    scales = torch.zeros(n if block == "row" else _ceil(n), _ceil(d), dtype=torch.float64, device=x.device)
    high = 1 if block == "row" else BLOCK
    for j in range(_ceil(d)):
        piece = x[:, j * BLOCK:(j + 1) * BLOCK].double()
        most = piece.abs().amax(dim=1)
        if high > 1:
            most = torch.stack([part.max() for part in most.split(high)])
        scales[:, j] = most.clamp(min=SMALLEST) / LARGEST
        y = piece / scales[:, j].float().double().repeat_interleave(high)[:n, None]
        # e4m3: three bits after the leading one, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, j * BLOCK:j * BLOCK + piece.shape[1]] = torch.round(y / step) * step
    return out, scales


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "product":
        return _expand(s["a"], s["a_scale"]) @ _expand(s["b"], s["b_scale"]).t()
    if kind == "grad":
        g, gs = _exact_scales(s["g"], "row")
        gt, gts = _exact_scales(s["g"].t(), "row")
        g = g * gs.float().double().repeat_interleave(BLOCK, dim=1)
        gt = gt * gts.float().double().repeat_interleave(BLOCK, dim=1)
        return g @ _expand(s["wt"], s["wt_scale"]).t(), gt @ _expand(s["xt"], s["xt_scale"]).t()
    if kind == "quantize":
        found = _exact_scales(s["x"], case["block"])
        if not case["transpose"]:
            return found
        if case["block"] == "row":
            return found + _exact_scales(s["x"].t(), "row")
        n, d = s["x"].shape
        turned = torch.zeros(d, _ceil(n) * BLOCK, dtype=torch.float64, device="cuda")
        turned[:, :n] = found[0][:, :d].t()
        return found + (turned, found[1].t())
    x = s["scores"]
    if kind == "top":
        values = x.double().sort(dim=1, descending=True).values[:, :case["k"]]
        short = case["k"] - values.shape[1]
        values = torch.nn.functional.pad(values, (0, short), value=-math.inf)
        return values, None, torch.logsumexp(x.double() / case["temperature"], dim=1)
    losses, grads = [], []
    t = case["temperature"]
    for i in range(0, x.shape[0], 256):
        z = x[i:i + 256].double() / t
        ids, val = s["ids"][i:i + 256].long(), s["values"][i:i + 256].double() / t
        there = (ids >= 0) & (ids < z.shape[1]) & (val > -math.inf)
        q = torch.log_softmax(z, dim=1)
        # the teacher's distribution over all columns, what it does not list apart
        if s["lse"] is None:
            p = torch.softmax(val.masked_fill(~there, -math.inf), dim=1)
        else:
            p = (val - s["lse"][i:i + 256].double()[:, None]).exp()
        p = torch.where(there, p, torch.zeros_like(p))
        dense = torch.zeros_like(z)
        dense.scatter_add_(1, ids.clamp(min=0), p)
        held = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), there.double()) > 0
        term = torch.where(dense > 0, dense * (dense.log() - q), torch.zeros_like(q)).sum(dim=1)
        grad = q.exp() * dense.sum(dim=1, keepdim=True) - dense
        if s["lse"] is not None:
            rest_q = torch.logsumexp(q.masked_fill(held, -math.inf), dim=1, keepdim=True)
            rest_p = torch.where(rest_q > -math.inf, (1 - dense.sum(dim=1, keepdim=True)).clamp(min=0),
                                 torch.zeros_like(rest_q))
            term = term + torch.where(rest_p > 0, rest_p * (rest_p.log() - rest_q), torch.zeros_like(rest_p))[:, 0]
            inside = torch.where(held | (rest_p == 0), torch.zeros_like(q), (q - rest_q).exp())
            grad = grad + rest_p * (q.exp() - inside)
        full = there.any(dim=1) & (z.amax(dim=1) > -math.inf)
        losses.append(torch.where(full, term, torch.zeros_like(term)))
        grad = grad * (s["weight"][i:i + 256].double() / t)[:, None]
        grads.append(torch.where(full[:, None], grad, torch.zeros_like(grad)))
    return torch.cat(losses), torch.cat(grads)
