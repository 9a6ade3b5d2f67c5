"""The operators that come after a quantization, measured: what a user runs on a packed model next.

    adapters    low-rank adapters of many requests beside a shared projection in the packed format: `forward` from one
                token to long prompts, and `backward`
    checkpoint  activations kept in 8 bits for the backward pass: `save` and `restore`, and the weight gradient from them
    loss        softmax cross entropy of a linear head over a large vocabulary without the logits, and its gradient

With `own` false, run() computes each operator in its plain form: elementary torch operations in 32 bits, rounded
once at the end.  With `own` true it makes the calls of cdclq.adapters, cdclq.checkpoint and cdclq.loss.
"""
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 128  # columns of a checkpoint that share a scale


def _cdclq():
    path = os.path.join(os.getcwd(), "cdcl-gptq_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import cdclq.adapters
    import cdclq.checkpoint
    import cdclq.loss

    return cdclq


# ---- cases ---------------------------------------------------------------------------------------------------------

def _projection(name, op, t, d_in, d_out, bits, group, n, r, dtype, wide=0, bare=0.0, kept=False):
    """wide: every wide-th column group has 8 bits (a skeleton); bare: share of tokens without an adapter; kept: the
    backward pass reads an 8-bit checkpoint of x."""
    c = {"op": op, "t": t, "d_in": d_in, "d_out": d_out, "bits": bits, "group": group, "adapters": n, "rank": r,
         "dtype": dtype, "wide": wide, "bare": bare, "kept": kept}
    return dict(c, name=name) if name else c


def _head(name, op, t, d, v, dtype, unlabelled=0.0, frozen=False):
    """unlabelled: share of tokens without a label; frozen: the head's weight gets no gradient."""
    c = {"op": op, "t": t, "d": d, "v": v, "dtype": dtype, "unlabelled": unlabelled, "frozen": frozen}
    return dict(c, name=name) if name else c


def _kept(name, op, t, d, dtype, d_out=0):
    c = {"op": op, "t": t, "d": d, "dtype": dtype, "d_out": d_out}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's next token through an attention projection (3 bits, groups of 128): latency
        _projection("decode 1", "forward", 1, 2048, 2048, 3, 128, 4, 16, "bf16"),
        # a decode batch, every request with its own adapter, through a wide up projection (4 bits, groups of 64)
        _projection("decode 12", "forward", 12, 4096, 11008, 4, 64, 12, 16, "f16"),
        # a ragged prompt batch through a down projection whose skeleton groups have 8 bits, some requests bare
        _projection("prompts 333", "forward", 333, 5632, 2048, 3, 128, 7, 8, "bf16", wide=16, bare=0.25),
        # a training or prefill batch through an attention projection
        _projection("batch 4096", "forward", 4096, 4096, 4096, 4, 64, 8, 32, "bf16"),
        # the backward pass of one fine-tuning step: x from an 8-bit checkpoint
        _projection("backward 2048", "backward", 2048, 2048, 5632, 3, 128, 1, 16, "bf16", kept=True),
        # the backward pass of several users' adapters trained together, x in full
        _projection("backward 4100", "backward", 4100, 4096, 4096, 4, 64, 6, 64, "f16", bare=0.1),
        # an activation saved and restored: of one short prompt, and of a training batch
        _kept("kept 300", "keep", 300, 2048, "f16"),
        _kept("kept 16384", "keep", 16384, 4096, "bf16"),
        # the weight gradient of a dense layer from the checkpoint of its input
        _kept("weight gradient 4096", "weight_grad", 4096, 2048, "bf16", 5632),
        # the loss of a few answers over a vocabulary that is not a round number (evaluation)
        _head("loss 57", "loss", 57, 2048, 50257, "bf16", unlabelled=0.2),
        # the end of a training step of adapters: the head is frozen, half of the tokens are prompt
        _head("step 2048 frozen", "step", 2048, 4096, 32000, "bf16", unlabelled=0.5, frozen=True),
        # the end of a training step that also trains the head
        _head("step 8191", "step", 8191, 2048, 32000, "f16", unlabelled=0.05),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["forward", "forward", "forward", "backward", "keep", "weight_grad", "loss", "step"])
    dtype = rng.choice(["bf16", "f16"])
    if op in ("forward", "backward"):
        d_in, d_out = 8 * _log(rng, 32, 1376), 8 * _log(rng, 32, 1376)
        if rng.random() < 0.3:
            d_out -= rng.randint(1, 7)
        group = rng.choice([32, 64, 128, 256, 0])
        t = _log(rng, 1, 4096) if op == "forward" else _log(rng, 16, 4096)
        while t * d_in * d_out > 4096 * 4096 * 4096 // (1 if op == "forward" else 2):
            t = t * 2 // 3 + 1
        return _projection(None, op, t, d_in, d_out, rng.choice([2, 3, 3, 4, 4, 8]), group, rng.choice([1, 2, 5, 16, 32]),
                           rng.choice([4, 8, 16, 24, 32, 64]), dtype, wide=rng.choice([0, 0, 8]) if group else 0,
                           bare=rng.choice([0.0, 0.3]), kept=op == "backward" and rng.random() < 0.5)
    if op == "keep":
        return _kept(None, op, _log(rng, 1, 16384), _log(rng, 64, 4096), rng.choice(["bf16", "f16", "f32"]))
    if op == "weight_grad":
        return _kept(None, op, _log(rng, 16, 4096), _log(rng, 64, 4096), dtype, _log(rng, 64, 4096))
    t, d, v = _log(rng, 1, 8192), 8 * _log(rng, 16, 512), _log(rng, 1000, 130000)
    while t * d * v > 8191 * 2048 * 32000:
        t = t * 2 // 3 + 1
    return _head(None, op, t, d, v, dtype, rng.choice([0.0, 0.1, 0.5]), rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------------------------------------------

def _columns(case):
    """Bits of each column group, and the group size."""
    g = case["group"] if 0 < case["group"] < case["d_in"] else case["d_in"]
    ng = -(-case["d_in"] // g)
    return [8 if case["wide"] and i % case["wide"] == 0 else case["bits"] for i in range(ng)], g


def _normal(shape, dtype, gen, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen).to(dtype)


def _tokens_adapters(case, gen):
    """The adapter of each token: requests of random lengths, each with one adapter or, as -1, none."""
    t, n = case["t"], case["adapters"]
    if t <= 32:  # a decode batch: every token is a request
        ids = torch.arange(t, device="cuda") % n
    else:
        cuts = torch.rand(t, generator=gen, device="cuda") < 1.0 / max(8.0, t / (2.0 * n))
        ids = torch.cumsum(cuts.long(), 0) % n
    lonely = torch.rand(t, generator=gen, device="cuda") < case["bare"]
    if t > 32:
        lonely = lonely[ids * 0 + torch.cumsum(cuts.long(), 0)]
    return torch.where(lonely, torch.full_like(ids, -1), ids).int()


def _prepare_projection(case, gen):
    t, d_in, d_out, n, r = (case[k] for k in ("t", "d_in", "d_out", "adapters", "rank"))
    dtype = DTYPES[case["dtype"]]
    gbits, g = _columns(case)
    widths = [min(g, d_in - i * g) for i in range(len(gbits))]
    row_bytes = (sum(b * w for b, w in zip(gbits, widths)) + 7) // 8
    bits = torch.tensor(gbits, device="cuda")
    half = (2 ** (bits - 1)).float()
    # weights of about 1 / sqrt(d_in), zero points around the middle of the grid
    spread = torch.rand(d_out, len(gbits), generator=gen, device="cuda") + 0.5
    s = {"case": case, "gsize": g, "index": _tokens_adapters(case, gen)}
    s["qweight"] = torch.randint(0, 256, (d_out, row_bytes), generator=gen, device="cuda", dtype=torch.uint8)
    s["scales"] = (spread * (1.7 / d_in ** 0.5) / half).half()
    noise = torch.randint(-1, 2, (d_out, len(gbits)), generator=gen, device="cuda")
    s["qzeros"] = (half.long() + noise).clamp(min=0).to(torch.uint8)
    s["perm"] = torch.randperm(d_in, generator=gen, device="cuda").int()
    s["gbits"] = bits.to(torch.uint8)
    s["a"] = _normal((n, r, d_in), dtype, gen, d_in ** -0.5)
    s["b"] = _normal((n, d_out, r), dtype, gen, 0.5 * r ** -0.5)
    s["scale"] = torch.rand(n, generator=gen, device="cuda") + 0.5
    s["x"] = _normal((t, d_in), dtype, gen)
    if case["op"] == "backward":
        s["dy"] = _normal((t, d_out), dtype, gen, 0.1)
        s["u"] = _down(s["x"].float(), s["a"], s["index"]).to(dtype)  # what the forward pass kept
        if case["kept"]:
            s["codes"], s["code_scales"] = _save(s["x"])
            del s["x"]
    if own:
        s["projection"] = _cdclq().adapters.PackedProjection(s["qweight"], s["scales"], s["qzeros"], s["perm"], s["gbits"], g)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("forward", "backward"):
        return _prepare_projection(case, gen)
    dtype, t, d = DTYPES[case["dtype"]], case["t"], case["d"]
    s = {"case": case}
    if case["op"] in ("keep", "weight_grad"):
        # activations whose channels have very different ranges
        ranges = torch.exp(torch.empty(d, device="cuda").normal_(0.0, 1.0, generator=gen))
        s["x"] = (_normal((t, d), torch.float32, gen) * ranges).to(dtype)
        if case["op"] == "weight_grad":
            s["codes"], s["code_scales"] = _save(s.pop("x"))
            s["dy"] = _normal((t, case["d_out"]), dtype, gen, 0.1)
        return s
    s["h"] = _normal((t, d), dtype, gen)
    s["w"] = _normal((case["v"], d), dtype, gen, 2.5 * d ** -0.5)
    s["target"] = torch.randint(0, case["v"], (t,), generator=gen, device="cuda")
    s["target"][torch.rand(t, generator=gen, device="cuda") < case["unlabelled"]] = -100
    # the mean's gradient, under a loss scale as half precision needs it
    s["dloss"] = torch.full((t,), (1.0 if case["dtype"] == "bf16" else 4096.0) / t, device="cuda")
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _dequantize(s):
    """The packed weight in 32 bits, original column order: LSB-first bit streams of mixed widths."""
    d_in = s["perm"].numel()
    width = s["gbits"].long().repeat_interleave(s["gsize"])[:d_in]
    off = torch.cumsum(width, 0) - width
    byte, shift = off // 8, (off % 8).int()
    last = s["qweight"].shape[1] - 1
    pair = s["qweight"][:, byte].int() | (s["qweight"][:, (byte + 1).clamp(max=last)].int() << 8)
    code = (pair >> shift) & ((1 << width.int()) - 1)
    col = torch.arange(d_in, device="cuda") // s["gsize"]
    w = s["scales"].float()[:, col] * (code.float() - s["qzeros"].float()[:, col])
    out = torch.empty_like(w)
    out[:, s["perm"].long()] = w
    return out


def _mask(index, n):
    return (index[:, None] == torch.arange(n, device="cuda")).float()


def _down(x, a, index):
    """x_t A_i^T with the adapter i of each token; zero without one."""
    n, r, d = a.shape
    u = (x @ a.float().reshape(n * r, d).t()).reshape(-1, n, r)
    return (u * _mask(index, n)[:, :, None]).sum(1)


def _spread(u, index, n):
    """[t, n * r]: u in the columns of the token's adapter, zero elsewhere."""
    return (u[:, None, :] * _mask(index, n)[:, :, None]).reshape(u.shape[0], -1)


def _save(x):
    t, d = x.shape
    pad = torch.nn.functional.pad(x.float(), (0, -d % BLOCK)).reshape(t, -1, BLOCK)
    top = pad.abs().amax(2)
    scale = top / torch.full_like(top, 127.0)
    codes = torch.round(pad / torch.where(scale > 0, scale, torch.ones_like(scale))[:, :, None]).clamp(-127, 127)
    return codes.reshape(t, -1)[:, :d].to(torch.int8).contiguous(), scale


def _restore(codes, scales):
    return codes.float() * scales.repeat_interleave(BLOCK, 1)[:, : codes.shape[1]]


def _plain_forward(s):
    n, r, d_in = s["a"].shape
    x = s["x"].float()
    u = _down(x, s["a"], s["index"])
    y = x @ _dequantize(s).t()
    up = (s["b"].float() * s["scale"][:, None, None]).permute(0, 2, 1).reshape(n * r, -1)
    y = y + _spread(u, s["index"], n) @ up
    return {"y": y.to(s["x"].dtype), "u": u.to(s["x"].dtype)}


def _plain_backward(s):
    n, r, d_in = s["a"].shape
    dt, dy = s["dy"].dtype, s["dy"].float()
    x = _restore(s["codes"], s["code_scales"]) if "codes" in s else s["x"].float()
    scaled = s["b"].float() * s["scale"][:, None, None]
    v = (dy @ scaled.permute(1, 0, 2).reshape(-1, n * r)).reshape(-1, n, r) * _mask(s["index"], n)[:, :, None]
    v = v.reshape(-1, n * r)
    dx = dy @ _dequantize(s) + v @ s["a"].float().reshape(n * r, d_in)
    da = (v.t() @ x).reshape(n, r, d_in)
    db = (_spread(s["u"].float(), s["index"], n).t() @ dy).reshape(n, r, -1).transpose(1, 2) * s["scale"][:, None, None]
    return {"dx": dx.to(dt), "da": da.to(dt), "db": db.to(dt)}


def _plain_loss(s):
    logits = s["h"].float() @ s["w"].float().t()
    top = logits.amax(1)
    lse = top + torch.log(torch.exp(logits - top[:, None]).sum(1))
    labelled = s["target"] >= 0
    at = torch.gather(logits, 1, s["target"].clamp(min=0)[:, None])[:, 0]
    return logits, lse, labelled, torch.where(labelled, lse - at, torch.zeros_like(lse))


def _plain_step(s):
    logits, lse, labelled, loss = _plain_loss(s)
    g = torch.exp(logits - lse[:, None])
    g[torch.arange(g.shape[0], device="cuda"), s["target"].clamp(min=0)] -= 1.0
    g = g * torch.where(labelled, s["dloss"], torch.zeros_like(lse))[:, None]
    out = {"loss": loss, "dh": (g @ s["w"].float()).to(s["h"].dtype)}
    if not s["case"]["frozen"]:
        out["dw"] = (g.t() @ s["h"].float()).to(s["w"].dtype)
    return out


def _plain(s):
    op = s["case"]["op"]
    if op == "forward":
        return _plain_forward(s)
    if op == "backward":
        return _plain_backward(s)
    if op == "keep":
        codes, scales = _save(s["x"])
        return {"values": _restore(codes, scales).to(s["x"].dtype), "scales": scales}
    if op == "weight_grad":
        return {"dw": (s["dy"].float().t() @ _restore(s["codes"], s["code_scales"])).to(s["dy"].dtype)}
    if op == "loss":
        _, lse, _, loss = _plain_loss(s)
        return {"loss": loss, "lse": lse}
    return _plain_step(s)


# ---- the framework's calls -----------------------------------------------------------------------------------------

def _calls(s):
    q, case = _cdclq(), s["case"]
    op = case["op"]
    if op == "forward":
        y, u = q.adapters.forward(s["x"], s["projection"], s["a"], s["b"], s["scale"], s["index"], keep=True)
        return {"y": y, "u": u}
    if op == "backward":
        x = q.checkpoint.Checkpoint(s["codes"], s["code_scales"], s["dy"].dtype) if case["kept"] else s["x"]
        dx, da, db = q.adapters.backward(s["dy"], x, s["u"], s["projection"], s["a"], s["b"], s["scale"], s["index"])
        return {"dx": dx, "da": da, "db": db}
    if op == "keep":
        c = q.checkpoint.save(s["x"])
        return {"values": q.checkpoint.restore(c), "scales": c.scales}
    if op == "weight_grad":
        return {"dw": q.checkpoint.weight_grad(s["dy"], q.checkpoint.Checkpoint(s["codes"], s["code_scales"], s["dy"].dtype))}
    loss, lse = q.loss.linear_cross_entropy(s["h"], s["w"], s["target"])
    if op == "loss":
        return {"loss": loss, "lse": lse}
    dh, dw = q.loss.linear_cross_entropy_backward(s["h"], s["w"], s["target"], lse, s["dloss"], need_dw=not case["frozen"])
    return {"loss": loss, "dh": dh} if case["frozen"] else {"loss": loss, "dh": dh, "dw": dw}


def run(state):
    return _calls(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("forward", "backward"):
        t, k, m, n, r = (case[x] for x in ("t", "d_in", "d_out", "adapters", "rank"))
        gbits, g = _columns(case)
        packed = m * (sum(b * min(g, k - i * g) for i, b in enumerate(gbits)) + 7) // 8 + 3 * m * len(gbits) + 4 * k
        used = min(n, t)
        adapters = 2 * used * r * (k + m) + 4 * n + 4 * t
        if op == "forward":
            return {"bytes": packed + adapters + 2 * t * (k + m + r), "flops": 2 * t * k * m + 2 * t * r * (k + m)}
        x = t * k + 4 * t * -(-k // BLOCK) if case["kept"] else 2 * t * k
        grads = 2 * n * r * (k + m)
        return {"bytes": packed + adapters + grads + x + 2 * t * (k + m + r), "flops": 2 * t * k * m + 4 * t * r * (k + m)}
    t, d, size = case["t"], case["d"], 4 if case["dtype"] == "f32" else 2
    kept = t * d + 4 * t * -(-d // BLOCK)
    if op == "keep":
        return {"bytes": 2 * (size * t * d + kept), "flops": 4 * t * d}  # the 8 bits are written, and read back later
    if op == "weight_grad":
        return {"bytes": kept + 2 * t * case["d_out"] + 2 * d * case["d_out"], "flops": 2 * t * d * case["d_out"]}
    v = case["v"]
    if op == "loss":
        return {"bytes": 2 * (t * d + v * d) + 16 * t, "flops": 2 * t * d * v}
    # without the logits they are computed a second time
    return {"bytes": 2 * (2 * t * d + (1 if case["frozen"] else 2) * v * d) + 16 * t,
            "flops": (6 if case["frozen"] else 8) * t * d * v}


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------

def _exact_weight(s):
    gbits, g = _columns(s["case"])
    d_out, d_in = s["qweight"].shape[0], s["case"]["d_in"]
    w = torch.zeros(d_out, d_in, dtype=torch.float64, device="cuda")
    stream = (s["qweight"][:, :, None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
    stream = stream.reshape(d_out, -1)
    at = 0
    for i, b in enumerate(gbits):
        cols = s["perm"][i * g:(i + 1) * g].long()
        part = stream[:, at:at + b * cols.numel()].reshape(d_out, cols.numel(), b).double()
        code = part @ (2.0 ** torch.arange(b, device="cuda", dtype=torch.float64))
        w[:, cols] = s["scales"][:, i:i + 1].double() * (code - s["qzeros"][:, i:i + 1].double())
        at += b * cols.numel()
    return w


def _exact_kept(s):
    x = s["codes"].double()
    for i in range(s["code_scales"].shape[1]):
        x[:, i * BLOCK:(i + 1) * BLOCK] *= s["code_scales"][:, i:i + 1].double()
    return x


def _exact_projection(s):
    case, w = s["case"], _exact_weight(s)
    n = case["adapters"]
    if case["op"] == "forward":
        x = s["x"].double()
        y = x @ w.t()
        u = torch.zeros(case["t"], case["rank"], dtype=torch.float64, device="cuda")
        for i in range(n):
            rows = (s["index"] == i).nonzero()[:, 0]
            u[rows] = x[rows] @ s["a"][i].double().t()
            y[rows] += s["scale"][i].double() * (u[rows] @ s["b"][i].double().t())
        return {"y": y, "u": u}
    x, dy, u = _exact_kept(s) if case["kept"] else s["x"].double(), s["dy"].double(), s["u"].double()
    dx = dy @ w
    da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for i in range(n):
        rows = (s["index"] == i).nonzero()[:, 0]
        k = s["scale"][i].double()
        back = k * (dy[rows] @ s["b"][i].double())
        dx[rows] += back @ s["a"][i].double()
        da[i] = back.t() @ x[rows]
        db[i] = k * (dy[rows].t() @ u[rows])
    return {"dx": dx, "da": da, "db": db}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("forward", "backward"):
        return _exact_projection(s)
    if op == "keep":
        d = case["d"]
        scales = torch.stack([s["x"][:, i:i + BLOCK].double().abs().amax(1) for i in range(0, d, BLOCK)], 1) / 127
        x = s["x"].double()
        for i in range(scales.shape[1]):  # the nearest multiple of the block's scale
            x[:, i * BLOCK:(i + 1) * BLOCK] = torch.round(x[:, i * BLOCK:(i + 1) * BLOCK] / scales[:, i:i + 1]) * scales[:, i:i + 1]
        return {"values": x, "scales": scales}
    if op == "weight_grad":
        return {"dw": s["dy"].double().t() @ _exact_kept(s)}
    h, w, rows = s["h"].double(), s["w"].double(), torch.arange(case["t"], device="cuda")
    loss, lse, dh = [], [], []
    dw = torch.zeros_like(w) if op == "step" and not case["frozen"] else None
    for some in rows.split(2048):
        logp = h[some] @ w.t()
        norm = torch.logsumexp(logp, 1)
        logp -= norm[:, None]
        label = s["target"][some]
        has = label >= 0
        lse.append(norm)
        loss.append(torch.where(has, -logp[torch.arange(some.numel(), device="cuda"), label.clamp(min=0)], 0.0))
        if op == "step":
            g = logp.exp_()
            g[torch.arange(some.numel(), device="cuda"), label.clamp(min=0)] -= 1
            g *= (s["dloss"][some].double() * has)[:, None]
            dh.append(g @ w)
            if dw is not None:
                dw += g.t() @ h[some]
    if op == "loss":
        return {"loss": torch.cat(loss), "lse": torch.cat(lse)}
    out = {"loss": torch.cat(loss), "dh": torch.cat(dh)}
    if dw is not None:
        out["dw"] = dw
    return out
