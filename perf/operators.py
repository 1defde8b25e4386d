"""Timing cases of the language-model operators: the fully connected layer with its activation and residual sum,
the softmax loss over a large vocabulary that never stores its logits, and the AdamW step over many tensors.

`own` chooses between the operators' plain form (elementary torch operations in 32 bits) and the framework's calls.
"""
import math

import torch

own = False

BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.95, 1e-8, 3e-4, 0.1
BLOCK = 256          # elements that share one scale where the optimizer's states are held in 8 bits
ARENA = 256          # tensors of the optimizer's arena start at a multiple of this many elements
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

_runtime = None


def _rt():
    """The framework's runtime, launching on torch's default stream."""
    global _runtime
    if _runtime is None:
        from swcompiler_amd.hip import runtime
        _runtime = runtime()
        _runtime.use_default_stream()
    return _runtime


# ------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decoder through a 4096-wide layer: the weights are read once, latency counts
        dict(name="fc token", op="fc", dtype="bf16", m=1, n=4096, k=4096, act="silu", bias=True, residual=True),
        # a ragged handful of sequences, widths that are no multiple of anything
        dict(name="fc ragged", op="fc", dtype="bf16", m=333, n=1411, k=1003, act="gelu", bias=True, residual=False),
        # a training batch through the widening layer of a block
        dict(name="fc batch", op="fc", dtype="bf16", m=4096, n=16384, k=4096, act="gelu_tanh", bias=True, residual=True),
        # the framework's own type at its wide MLP's size
        dict(name="fc batch f32", op="fc", dtype="f32", m=2048, n=4096, k=4096, act="gelu", bias=True, residual=True),
        # gradients of the widening layer
        dict(name="fc grad", op="fc_grad", dtype="bf16", m=4096, n=16384, k=4096, act="gelu_tanh", bias=True),
        # gradients of a small fp32 layer
        dict(name="fc grad f32", op="fc_grad", dtype="f32", m=512, n=1024, k=784, act="silu", bias=True),
        # scoring a short text: losses only, a thousand classes as the image models have
        dict(name="loss small f32", op="loss", dtype="f32", m=64, n=1000, k=512, bias=True, left_out=0.0, grad=False),
        # a training step's loss and gradients over a vocabulary of odd length, prompt tokens left out
        dict(name="loss ragged", op="loss", dtype="bf16", m=1999, n=50257, k=1024, bias=False, left_out=0.3, grad=True),
        # the largest step: 8192 tokens against a vocabulary of 128256
        dict(name="loss batch", op="loss", dtype="bf16", m=8192, n=128256, k=4096, bias=False, left_out=0.0, grad=True),
        # an optimizer step of the 784-512-10 MLP
        dict(name="adamw small", op="adamw", bits=32, grads="f32", inner=784, hidden=512, layers=1, out=10, copy=False),
        # a language model's step: bf16 gradients and bf16 weights for the products, 32-bit states
        dict(name="adamw batch", op="adamw", bits=32, grads="bf16", inner=4096, hidden=4096, layers=8, out=32000, copy=True),
        # the same with states in 8 bits
        dict(name="adamw 8 bits", op="adamw", bits=8, grads="bf16", inner=2048, hidden=2048, layers=8, out=32000, copy=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """a layer's width: most often a multiple of 64, sometimes any number"""
    w = _log(rng, low, high)
    return w if rng.random() < 0.25 else max(64, w // 64 * 64)


def draw(rng):
    op = rng.choice(["fc", "fc_grad", "loss", "loss", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("fc", "fc_grad"):
        top = 16384 if dtype == "bf16" else 4096
        c = dict(op=op, dtype=dtype, m=_log(rng, 1, 4096), n=_width(rng, 64, top), k=_width(rng, 64, min(top, 8192)),
                 act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7)
        if op == "fc":
            c["residual"] = rng.random() < 0.5
        return c
    if op == "loss":
        big = dtype == "bf16"
        return dict(op=op, dtype=dtype, m=_log(rng, 1, 8192 if big else 2048), n=_log(rng, 1000, 128256 if big else 32768),
                    k=_width(rng, 64, 4096 if big else 1024), bias=rng.random() < 0.3,
                    left_out=rng.choice([0.0, 0.0, 0.2, 0.6]), grad=rng.random() < 0.7)
    return dict(op=op, bits=rng.choice([8, 32]), grads=rng.choice(["bf16", "f32"]), inner=_log(rng, 64, 4096),
                hidden=_log(rng, 64, 2048), layers=rng.randint(1, 8), out=_log(rng, 10, 32000), copy=rng.random() < 0.7)


def _sizes(case):
    """the tensors of an MLP of `layers` hidden layers: weight and bias of each, input first"""
    i, h, o = case["inner"], case["hidden"], case["out"]
    return [i * h, h] + [h * h, h] * (case["layers"] - 1) + [h * o, o]


def _starts(sizes):
    at, starts = 0, []
    for s in sizes:
        starts.append(at)
        at += -(-s // ARENA) * ARENA
    return starts, at


def work(case):
    if case["op"] in ("fc", "fc_grad"):
        m, n, k, e = case["m"], case["n"], case["k"], 2 if case["dtype"] == "bf16" else 4
        if case["op"] == "fc":
            values = m * k + k * n + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
            return {"bytes": e * values, "flops": 2 * m * n * k}
        values = 2 * m * k + 2 * k * n + m * n * (1 if case["act"] == "none" else 2) + (n if case["bias"] else 0)
        return {"bytes": e * values, "flops": 4 * m * n * k}
    if case["op"] == "loss":
        m, n, k, e = case["m"], case["n"], case["k"], 2 if case["dtype"] == "bf16" else 4
        rows = max(1, round(m * (1 - case["left_out"])))   # rows that are left out need no products
        once = m * k + k * n + (n if case["bias"] else 0)
        return {"bytes": e * once * (2 if case["grad"] else 1) + 12 * m, "flops": (6 if case["grad"] else 2) * rows * n * k}
    total = sum(_sizes(case))
    state = 8 * 2 if case["bits"] == 32 else 2 * 2
    per = 8 + (2 if case["grads"] == "bf16" else 4) + state + (2 if case["copy"] else 0)
    return {"bytes": per * total, "flops": 16 * total}


# ------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dtype)

    s = dict(case)
    if case["op"] in ("fc", "fc_grad", "loss"):
        m, n, k, dt = case["m"], case["n"], case["k"], TYPES[case["dtype"]]
        s["a"] = normal(m, k, dtype=dt)
        s["b"] = normal(k, n, scale=k ** -0.5, dtype=dt)
        s["bias_v"] = normal(n, scale=0.3, dtype=dt) if case["bias"] else None
        if case["op"] == "fc":
            s["res"] = normal(m, n, dtype=dt) if case["residual"] else None
        elif case["op"] == "fc_grad":
            s["dc"] = normal(m, n, dtype=dt)
            s["pre"] = normal(m, n, dtype=dt) if case["act"] != "none" else None
        else:
            labels = torch.randint(0, n, (m,), generator=gen, device="cuda")
            if case["left_out"]:
                labels[torch.rand(m, generator=gen, device="cuda") < case["left_out"]] = -1
            s["labels"] = labels.to(torch.int32)
        return s
    sizes = _sizes(case)
    starts, total = _starts(sizes)
    s["tensors"] = list(zip(starts, sizes))
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for at, size in s["tensors"]:
        inside[at:at + size] = True

    def arena(values):
        return values.mul_(inside)

    s["w"] = arena(normal(total, scale=0.02))
    s["g"] = arena(normal(total, scale=1e-3)).to(TYPES[case["grads"]])
    s["copy_v"] = s["w"].to(torch.bfloat16) if case["copy"] else None
    s["state"] = torch.zeros(8, dtype=torch.int32, device="cuda")
    s["state"][0] = 100
    mom = arena(normal(total, scale=3e-4))
    root = arena(normal(total, scale=1e-3).abs_())
    if case["bits"] == 32:
        s["mom"], s["var"] = mom, root.square()
        return s
    s["key"] = torch.cat([torch.arange(-(-size // ARENA) * ARENA, device="cuda") + t * 0x9E3779B9
                          for t, size in enumerate(sizes)]).bitwise_and_(0xFFFFFFFF)
    for name, value in (("mom", mom), ("var", root)):
        rows = value.view(-1, BLOCK)
        scale = rows.abs().amax(1) / 448
        s[name + "_scale"] = scale
        s[name] = (rows / scale.clamp(min=1e-30)[:, None]).to(torch.float8_e4m3fn).view(-1)
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _fc_plain(s):
    z = s["a"].float() @ s["b"].float()
    if s["bias_v"] is not None:
        z += s["bias_v"].float()
    c = _act(z, s["act"])
    if s["res"] is not None:
        c = c + s["res"].float()
    return {"c": c.to(s["a"].dtype)}


def _fc_grad_plain(s):
    dt = s["a"].dtype
    dz = s["dc"].float()
    if s["act"] != "none":
        dz = dz * _act_slope(s["pre"].float(), s["act"])
    out = {"da": (dz @ s["b"].float().t()).to(dt), "db": (s["a"].float().t() @ dz).to(dt)}
    if s["bias_v"] is not None:
        out["dbias"] = dz.sum(0).to(dt)
    return out


def _loss_plain(s):
    dt, labels = s["a"].dtype, s["labels"].long()
    counts = labels >= 0
    a, b = torch.where(counts[:, None], s["a"].float(), 0), s["b"].float()
    z = a @ b
    if s["bias_v"] is not None:
        z += s["bias_v"].float()
    top = z.amax(1)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
    picked = z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    row = torch.where(counts, lse - picked, 0)
    lse = torch.where(counts, lse, 0)
    out = {"loss": row.sum() / counts.sum().clamp(min=1), "row_loss": row, "lse": lse}
    if not s["grad"]:
        return out
    z = torch.exp(z - lse[:, None])
    z.scatter_add_(1, labels.clamp(min=0)[:, None], torch.full_like(lse, -1)[:, None])
    z = torch.where(counts[:, None], z, 0)
    out["da"], out["db"] = (z @ b.t()).to(dt), (a.t() @ z).to(dt)
    if s["bias_v"] is not None:
        out["dbias"] = z.sum(0).to(dt)
    return out


def _random20(key, step):
    """20 random bits of an element in a step: two multiply-and-shift rounds over its number and the step's"""
    x = (key + step * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return (x ^ (x >> 16)) >> 12


def _adamw_plain(s):
    s["state"][0] += 1
    t = s["state"][0].long()
    c1, c2 = ((1 / (1 - torch.pow(torch.tensor(b, dtype=torch.float64, device="cuda"), t))).float() for b in (BETA1, BETA2))
    g = s["g"].float()
    if s["bits"] == 32:
        mom, var = s["mom"], s["var"]
        mom.mul_(BETA1).add_(g * (1 - BETA1))
        var.mul_(BETA2).add_(g * g * (1 - BETA2))
    else:
        mom = (s["mom"].float().view(-1, BLOCK) * s["mom_scale"][:, None]).view(-1)
        root = (s["var"].float().view(-1, BLOCK) * s["var_scale"][:, None]).view(-1)
        mom = mom * BETA1 + g * (1 - BETA1)
        var = root * root * BETA2 + g * g * (1 - BETA2)
    s["w"].mul_(1 - LR * DECAY).sub_(LR * c1 * mom / (torch.sqrt(var * c2) + EPS))
    out = {"w": s["w"], "mom": s["mom"], "var": s["var"]}
    if s["copy_v"] is not None:
        s["copy_v"].copy_(s["w"])
        out["copy"] = s["copy_v"]
    if s["bits"] == 8:
        rows, roots = mom.view(-1, BLOCK), torch.sqrt(var).view(-1, BLOCK)
        s["mom_scale"].copy_(rows.abs().amax(1) / 448)
        s["var_scale"].copy_(roots.amax(1) / 448)
        # the mean to the nearest value; which side of a border it lies on is settled in 64 bits
        y = torch.where(s["mom_scale"][:, None] > 0, rows.double() / s["mom_scale"].double()[:, None], 0).clamp(-448, 448)
        s["mom"].copy_(y.float().view(-1))
        # the root of the variance up or down at random, a nonzero one never to zero
        y = torch.where(s["var_scale"][:, None] > 0, roots.double() / s["var_scale"].double()[:, None], 0).clamp(max=448)
        y = y.view(-1)
        step = torch.exp2(torch.frexp(y)[1].clamp(min=-5).double() - 4)
        q = torch.floor(y / step + _random20(s["key"], t).double() * 2.0 ** -20)
        s["var"].copy_((torch.where(y > 0, q.clamp(min=1), 0) * step).float())
        out["mom_scale"], out["var_scale"] = s["mom_scale"], s["var_scale"]
    return out


# --------------------------------------------------------------------------------------------- the framework's
def _fc_own(s):
    rt, a, b = _rt(), s["a"], s["b"]
    c = torch.empty(s["m"], s["n"], dtype=a.dtype, device="cuda")
    rt.matrixMatrixFCActAdd(a, b, s["bias_v"], s["act"], s["res"], out=c)
    return {"c": c}


def _fc_grad_own(s):
    rt, a, b = _rt(), s["a"], s["b"]
    out = {"da": torch.empty_like(a), "db": torch.empty_like(b)}
    if s["bias_v"] is not None:
        out["dbias"] = torch.empty_like(s["bias_v"])
    rt.matrixMatrixFCActAddGrad(s["dc"], a, b, s["pre"], s["act"], da=out["da"], db=out["db"], dbias=out.get("dbias"))
    return out


def _loss_own(s):
    rt, a, b = _rt(), s["a"], s["b"]
    out = {"loss": torch.empty((), device="cuda"), "row_loss": torch.empty(s["m"], device="cuda"),
           "lse": torch.empty(s["m"], device="cuda")}
    rt.matrixFCSoftmaxWithLoss(a, b, s["bias_v"], s["labels"], loss=out["loss"], row_loss=out["row_loss"], lse=out["lse"])
    if s["grad"]:
        out["da"], out["db"] = torch.empty_like(a), torch.empty_like(b)
        if s["bias_v"] is not None:
            out["dbias"] = torch.empty_like(s["bias_v"])
        rt.matrixFCSoftmaxWithLossGrad(a, b, s["bias_v"], s["labels"], out["lse"], da=out["da"], db=out["db"],
                                       dbias=out.get("dbias"))
    return out


def _adamw_own(s):
    rt = _rt()

    def parts(name):
        x = s[name]
        return None if x is None else [x[at:at + size] for at, size in s["tensors"]]

    def scales(name):
        return [s[name][at // BLOCK:at // BLOCK + -(-size // BLOCK)] for at, size in s["tensors"]]

    rt.adamwAdvance(s["state"], BETA1, BETA2)
    out = {"w": s["w"], "mom": s["mom"], "var": s["var"]}
    if s["bits"] == 8:
        rt.adamw8(parts("w"), parts("g"), parts("mom"), scales("mom_scale"), parts("var"), scales("var_scale"), s["state"],
                  LR, BETA1, BETA2, EPS, DECAY, copies=parts("copy_v"))
        out["mom_scale"], out["var_scale"] = s["mom_scale"], s["var_scale"]
    else:
        rt.adamw(parts("w"), parts("g"), parts("mom"), parts("var"), s["state"], LR, BETA1, BETA2, EPS, DECAY,
                 copies=parts("copy_v"))
    if s["copy_v"] is not None:
        out["copy"] = s["copy_v"]
    return out


def run(state):
    op = state["op"]
    if own:
        return {"fc": _fc_own, "fc_grad": _fc_grad_own, "loss": _loss_own, "adamw": _adamw_own}[op](state)
    return {"fc": _fc_plain, "fc_grad": _fc_grad_plain, "loss": _loss_plain, "adamw": _adamw_plain}[op](state)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _adamw_exact(s)
    a, b = s["a"].double(), s["b"].double()
    bias = s["bias_v"].double() if s["bias_v"] is not None else None
    if case["op"] == "fc":
        z = torch.addmm(bias, a, b) if bias is not None else torch.mm(a, b)
        c = _exact_act(z, case["act"])
        return {"c": c if s["res"] is None else torch.add(c, s["res"].double())}
    if case["op"] == "fc_grad":
        dz = s["dc"].double()
        if case["act"] != "none":
            pre = s["pre"].double().requires_grad_()
            dz, = torch.autograd.grad(_exact_act(pre, case["act"]), pre, dz)
        out = {"da": torch.mm(dz, b.t().contiguous()), "db": torch.mm(a.t().contiguous(), dz)}
        if bias is not None:
            out["dbias"] = torch.sum(dz, 0)
        return out
    rows = torch.nonzero(s["labels"] >= 0)[:, 0]     # by the definition, over the rows that count alone
    labels, a = s["labels"][rows].long(), a[rows]
    z = torch.addmm(bias, a, b) if bias is not None else torch.mm(a, b)
    lse = torch.logsumexp(z, 1)
    row = lse - z[torch.arange(len(rows), device="cuda"), labels]
    whole = torch.zeros(case["m"], dtype=torch.float64, device="cuda")
    out = {"loss": row.sum() / max(1, len(rows)), "row_loss": whole.index_copy(0, rows, row),
           "lse": whole.index_copy(0, rows, lse)}
    if case["grad"]:
        dz = torch.softmax(z, 1)
        del z
        dz[torch.arange(len(rows), device="cuda"), labels] -= 1
        da = torch.zeros(case["m"], case["k"], dtype=torch.float64, device="cuda")
        out["da"] = da.index_copy_(0, rows, torch.mm(dz, b.t().contiguous()))
        out["db"] = torch.mm(a.t().contiguous(), dz)
        if bias is not None:
            out["dbias"] = torch.sum(dz, 0)
    return out


def _exact_act(z, act):
    f = torch.nn.functional
    return {"none": lambda x: x, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda x: f.gelu(x, approximate="tanh"),
            "silu": f.silu}[act](z)


def _adamw_exact(s):
    t = int(s["state"][0]) + 1
    g, w = s["g"].double(), s["w"].double()
    if s["bits"] == 32:
        mom, var = s["mom"].double(), s["var"].double()
    else:
        mom = s["mom"].double() * s["mom_scale"].double().repeat_interleave(BLOCK)
        var = torch.square(s["var"].double() * s["var_scale"].double().repeat_interleave(BLOCK))
    mom, var = torch.lerp(g, mom, BETA1), torch.lerp(g * g, var, BETA2)
    w = w - LR * DECAY * w - LR * (mom / (1 - BETA1 ** t)) / (torch.sqrt(var / (1 - BETA2 ** t)) + EPS)
    out = {"w": w, "mom": mom, "var": var, "copy": w if s["copy_v"] is not None else None}
    if s["bits"] == 8:
        top = mom.abs().view(-1, BLOCK).max(1).values
        peak = var.view(-1, BLOCK).max(1).values.sqrt()
        out["mom_scale"], out["var_scale"] = top / 448, peak / 448
        y = torch.nan_to_num(mom.view(-1, BLOCK) * (448 / top)[:, None], nan=0.0).view(-1)
        grid = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        out["mom"] = torch.round(y / grid) * grid
        y = torch.nan_to_num(var.sqrt().view(-1, BLOCK) * (448 / peak)[:, None], nan=0.0).view(-1)
        grid = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
        x = torch.remainder(s["key"] + 0x85EBCA6B * t, 1 << 32)
        x = torch.remainder(torch.bitwise_xor(x, x // 65536) * 0x7FEB352D, 1 << 32)
        x = torch.bitwise_xor(x, x // 32768)
        x = torch.bitwise_and(x * 0x846CA68B, 0xFFFFFFFF)
        x = torch.bitwise_xor(x, x // 65536) // 4096
        up = torch.floor(y / grid + x.double() / 1048576)
        out["var"] = torch.where(y > 0, up.clamp(min=1), up) * grid
    return {k: v for k, v in out.items() if v is not None}
