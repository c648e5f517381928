"""Cases for the operators of a softmax-attention encoder's training step.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as the
framework offers it:

  * attention: ``ops.jagged_attention``, softmax attention of each head over the rows of its
    own sequence, alone (serving) or with the gradients of q, k and v (training);
  * layer_norm: ``ops.layer_norm`` over the last dimension, alone or with its gradients;
  * adamw8: one step of ``optim.FlatAdamW(state_bits=8)`` over a list of tensors.
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 64  # elements of a tensor that share one scale of an 8-bit moment
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.98), 1e-8, 1e-3
MASK = 0xFFFFFFFF


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one user's short history, served alone: latency counts
        attention("history of one user", 1, 37, 4, 4, 50, 50, "bf16", grad=False),
        # the ml-1m training batch (128 x 211, one head of 50) in the framework's default type,
        # its rows a buffer of full capacity behind the last sequence
        attention("ml-1m batch, training", 128, 211, 1, 1, 50, 50, "fp32", spare=True),
        # the ml-20m training batch (32 x 2059, one head of 256)
        attention("ml-20m batch, training", 32, 2059, 1, 1, 256, 256, "bf16"),
        # the same width as eight heads that share two key / value heads
        attention("shared heads, training", 24, 1499, 8, 2, 64, 64, "bf16"),
        # few long histories: little to spread over the chip but the rows themselves
        attention("long histories", 2, 8192, 4, 4, 128, 128, "bf16", grad=False),
        # the query rows of one retrieval batch
        norm("query rows", 128, 50, 50, "fp32", affine=False, grad=False),
        # the postprocessor on the ml-1m batch: the first 50 columns of wider rows
        norm("ml-1m rows, training", 27008, 50, 64, "fp32", affine=False),
        # the ml-20m batch's rows, with weight and bias
        norm("ml-20m rows, training", 65888, 256, 256, "bf16"),
        # wide hidden rows
        norm("wide rows, training", 20011, 4096, 4096, "bf16"),
        # the two-block encoder of the ml-1m configuration: many small tensors
        adamw("ml-1m encoder", 0, 50, 2, 211),
        # the eight-block encoder of the ml-20m width
        adamw("ml-20m encoder", 0, 256, 8, 2059),
        # the same with its item table
        adamw("ml-20m table and encoder", 131262, 256, 8, 2059),
    ]


def attention(name, batch, longest, heads, kv_heads, dim, dim_v, dtype, causal=True, grad=True, spare=False):
    return {"name": name, "op": "attention", "batch": batch, "longest": longest, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dim_v": dim_v, "dtype": dtype, "causal": causal, "grad": grad, "spare": spare}


def norm(name, rows, dim, row_stride, dtype, affine=True, grad=True):
    return {"name": name, "op": "layer_norm", "rows": rows, "dim": dim, "row_stride": row_stride, "dtype": dtype,
            "affine": affine, "grad": grad}


def adamw(name, items, dim, blocks, longest):
    return {"name": name, "op": "adamw8", "items": items, "dim": dim, "blocks": blocks, "longest": longest}


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("attention", "attention", "layer_norm", "adamw8"))
    while True:
        if op == "attention":
            kv = rng.choice((1, 1, 2, 3, 4))
            dim = rng.choice((rng.randint(8, 256), 50, 64, 128, 256))
            c = attention("", spread(1, 256), spread(2, 8192), kv * rng.choice((1, 1, 2, 4)), kv, dim,
                          rng.choice((dim, dim, rng.randint(8, 256))), rng.choice(("bf16", "bf16", "fp32")),
                          rng.random() < 0.8, rng.random() < 0.7, rng.random() < 0.3)
            full = c["batch"] * c["heads"] * c["longest"] ** 2
            most = work(listed()[2])["flops"]
            fits = full <= 5.4e8 and work(c)["flops"] <= (most if c["dtype"] == "bf16" else most / 8)
        elif op == "layer_norm":
            rows, dim = spread(1, 70000), spread(3, 8192)
            c = norm("", rows, dim, dim + rng.choice((0, 0, 0, 1, 14, 64)), rng.choice(("fp32", "bf16")),
                     rng.random() < 0.7, rng.random() < 0.7)
            fits = rows * dim <= 20011 * 4096
        else:
            c = adamw("", rng.choice((0, spread(100, 131262))), rng.choice((rng.randint(8, 256), 50, 64, 256)),
                      rng.randint(1, 8), spread(16, 2059))
            fits = True
        if fits:
            del c["name"]
            return c


def lengths_of(case):
    """The lengths of a case's sequences in ascending order: spread from a twentieth of the longest to the
    longest, an empty sequence and one of a single row among them where there are eight or more."""
    n, top = case["batch"], case["longest"]
    got = [max(1, round(top * (0.05 + 0.95 * (i + 0.5) / n))) for i in range(n - 1)] + [top]
    if n >= 8:
        got[0], got[1] = 0, 1
    return got


def shapes_of(case):
    """The parameters of an encoder of so many blocks (one head as wide as the rows), and of its item table."""
    d, n = case["dim"], case["longest"]
    return ([(case["items"], d)] if case["items"] else []) + [
        s for _ in range(case["blocks"]) for s in ((d, 4 * d), (d, d), (d,), (2 * n - 1,), (129,))]


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    state = {"case": case}
    if case["op"] == "attention":
        lens = torch.tensor(lengths_of(case))[torch.randperm(case["batch"], generator=torch.Generator().manual_seed(seed))]
        offsets = torch.zeros(case["batch"] + 1, dtype=torch.int64)
        offsets[1:] = lens.cumsum(0)
        rows = case["batch"] * case["longest"] if case["spare"] else int(offsets[-1])
        h, kv, d, dv = case["heads"], case["kv_heads"], case["dim"], case["dim_v"]
        # q, k and v are column slices of one projection's rows, as the encoder's are
        wide = (1.5 * randn(rows, h * d + kv * d + kv * dv)).to(TYPES[case["dtype"]])
        state["q"] = wide[:, :h * d].view(rows, h, d)
        state["k"] = wide[:, h * d:(h + kv) * d].view(rows, kv, d)
        state["v"] = wide[:, (h + kv) * d:].view(rows, kv, dv)
        state["offsets"] = offsets.to(DEVICE)
        state["longest"] = case["longest"]
        if case["grad"]:
            state["dout"] = randn(rows, h, dv).to(TYPES[case["dtype"]])
            state.update({n: state[n].detach().requires_grad_(True) for n in "qkv"})
    elif case["op"] == "layer_norm":
        rows, d, dt = case["rows"], case["dim"], TYPES[case["dtype"]]
        state["x"] = (2 * randn(rows, case["row_stride"]) + 0.5 * randn(rows, 1)).to(dt)[:, :d]
        state["weight"] = (1 + 0.2 * randn(d)) if case["affine"] else None
        state["bias"] = 0.1 * randn(d) if case["affine"] else None
        if case["grad"]:
            state["dy"] = randn(rows, d).to(dt)
            state.update({n: state[n].detach().requires_grad_(True) for n in ("x", "weight", "bias") if state[n] is not None})
    else:
        shapes = shapes_of(case)
        sizes = [math.prod(s) for s in shapes]
        padded = [-(-n // BLOCK) * BLOCK for n in sizes]
        params = [torch.nn.Parameter(0.02 * randn(*s)) for s in shapes]
        for p in params:
            # each tensor has gradients of a size of its own, its first axis' entries too
            p.grad = randn(*p.shape) * (10 ** (randn(p.shape[0], *[1] * (p.dim() - 1)) - 4))
        live = torch.cat([torch.arange(m, device=DEVICE) < n for n, m in zip(sizes, padded)])
        grads = torch.cat([torch.nn.functional.pad(p.grad.flatten(), (0, m - n)) for p, n, m in zip(params, sizes, padded)])
        # moments of a program that has taken a thousand steps, held in 8 bits
        state["exp_avg"], state["exp_avg_scale"] = held(0.3 * grads * randn(grads.numel()))
        state["exp_avg_sq"], state["exp_avg_sq_scale"] = held(grads.square() * (0.3 + randn(grads.numel()).square()) + 1e-14 * live)
        state.update(params=params, sizes=sizes, padded=padded, step=torch.full((1,), 1000.0, device=DEVICE))
    return state


def held(x):
    """(e4m3 values, power-of-two scale of each BLOCK) near x."""
    x = x.view(-1, BLOCK)
    scale = torch.exp2(torch.floor(torch.log2(x.abs().amax(1, keepdim=True).clamp(min=1e-28))) - 7)
    return (x / scale).to(torch.float8_e4m3fn).view(-1), scale.view(-1)


# ---------------------------------------------------------------- one pass

def run(state):
    return {"attention": run_attention, "layer_norm": run_norm, "adamw8": run_adamw}[state["case"]["op"]](state)


def run_attention(state):
    case = state["case"]
    q, k, v, offsets = (state[n] for n in ("q", "k", "v", "offsets"))
    if own:
        from mygenerativerecommenders_amd import ops
        out = ops.jagged_attention(q, k, v, offsets, causal=case["causal"])
        if not case["grad"]:
            return out
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), state["dout"])]
    with torch.no_grad():
        return plain_attention(q, k, v, offsets, state["longest"], case["causal"], state["dout"] if case["grad"] else None)


def plain_attention(q, k, v, offsets, longest, causal, dout):
    rows, h, d = q.shape
    kv, group, dev = k.shape[1], h // k.shape[1], q.device
    at = torch.arange(longest, device=dev)
    live = at < (offsets[1:] - offsets[:-1]).unsqueeze(1)
    index = (offsets[:-1].unsqueeze(1) + at).clamp(max=max(rows - 1, 0))
    row = torch.arange(rows, device=dev)
    owner = torch.searchsorted(offsets, row, right=True) - 1
    inside = owner < live.shape[0]
    owner = owner.clamp(max=live.shape[0] - 1)
    place = (row - offsets[owner]).clamp(0, longest - 1)

    def dense(x):  # (rows, heads, width) -> (batch, kv heads, group, longest, width), zero past a sequence's end
        x = x[index].float() * live[:, :, None, None]
        return x.view(*index.shape, kv, -1, x.shape[-1]).permute(0, 2, 3, 1, 4).contiguous()

    def jagged(x, dtype):
        x = x.permute(0, 3, 1, 2, 4).reshape(*index.shape, -1, x.shape[-1])
        return (x[owner, place] * inside[:, None, None]).to(dtype)

    qd, kd, vd = dense(q), dense(k), dense(v)
    sees = live[:, None, None, None, :] & live[:, None, None, :, None]
    if causal:
        sees = sees & (at <= at.unsqueeze(1))
    s = torch.matmul(qd, kd.transpose(-1, -2)) * d ** -0.5
    s = s.masked_fill(~sees, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    del s
    out = torch.matmul(p, vd)
    if dout is None:
        return jagged(out, q.dtype)
    g = dense(dout)
    ds = torch.matmul(g, vd.transpose(-1, -2))
    ds = p * (ds - (g * out).sum(-1, keepdim=True)) * d ** -0.5
    dq = torch.matmul(ds, kd)
    dk = torch.matmul(ds.transpose(-1, -2), qd).sum(2, keepdim=True)
    dv = torch.matmul(p.transpose(-1, -2), g).sum(2, keepdim=True)
    return [jagged(out, q.dtype), jagged(dq, q.dtype), jagged(dk, k.dtype), jagged(dv, v.dtype)]


def run_norm(state):
    case, x, w, b = state["case"], state["x"], state["weight"], state["bias"]
    if own:
        from mygenerativerecommenders_amd import ops
        y = ops.layer_norm(x, w, b, eps=1e-6)
        if not case["grad"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], state["dy"])]
    with torch.no_grad():
        xf = x.float()
        c = xf - xf.mean(-1, keepdim=True)
        r = torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-6)
        xh = c * r
        y = (xh * w + b if w is not None else xh).to(x.dtype)
        if not case["grad"]:
            return y
        dy = state["dy"].float()
        g = dy * w if w is not None else dy
        dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        return [y, dx.to(x.dtype)] + ([(dy * xh).sum(0), dy.sum(0)] if w is not None else [])


def run_adamw(state):
    params = state["params"]
    if own:
        opt = state.get("optimizer") or resumed(state)
        opt.step()
        held_now = opt.flat_state(0)
        return [[p.detach() for p in params],
                [held_now[n] for n in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale", "step")]]
    with torch.no_grad():
        sizes, padded = state["sizes"], state["padded"]
        p, g = (torch.cat([torch.nn.functional.pad(t.flatten(), (0, m - n)) for t, n, m in zip(ts, sizes, padded)])
                for ts in (params, [t.grad for t in params]))
        state["step"].add_(1)
        t = state["step"].double()
        m = decoded(state["exp_avg"], state["exp_avg_scale"]) * BETAS[0] + g * (1 - BETAS[0])
        v = decoded(state["exp_avg_sq"], state["exp_avg_sq_scale"]) * BETAS[1] + g * g * (1 - BETAS[1])
        size = (LR / (1 - BETAS[0] ** t)).float()
        root = torch.sqrt(1 - BETAS[1] ** t).float()
        p = p * (1 - LR * DECAY) - size * (m / (torch.sqrt(v) / root + EPS))
        live = [x[:n].view_as(t) for x, n, t in zip(p.split(padded), sizes, params)]
        torch._foreach_copy_([t.data for t in params], live)
        bits = random_bits(p.numel(), state["step"])
        state["exp_avg"], state["exp_avg_scale"] = rounded(m, bits & 0xFFFFF, False)
        state["exp_avg_sq"], state["exp_avg_sq_scale"] = rounded(v, bits >> 12, True)
        return [[t.detach() for t in params],
                [state[n] for n in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale", "step")]]


def resumed(state):
    """The optimizer of a program that goes on from a checkpoint with these moments."""
    from mygenerativerecommenders_amd.optim import FlatAdamW
    params = state["params"]
    opt = FlatAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=8)
    at = [sum(state["padded"][:i]) for i in range(len(params))]
    kept = opt.state_dict()
    kept["state"] = {i: {
        "step": state["step"],
        **{n: state[n][a:a + p.numel()].view(p.shape) for n in ("exp_avg", "exp_avg_sq")},
        **{n: state[n][a // BLOCK:(a + m) // BLOCK] for n in ("exp_avg_scale", "exp_avg_sq_scale")},
    } for i, (p, a, m) in enumerate(zip(params, at, state["padded"]))}
    opt.load_state_dict(kept)
    state["optimizer"] = opt
    return opt


def decoded(code, scale):
    return (code.float().view(-1, BLOCK) * scale.view(-1, 1)).view(-1)


def random_bits(n, step):
    """32 bits for each element: a hash of its place and of the step's number."""
    key = (step.to(torch.int64) * 0xA54FF53B) & MASK
    x = (torch.arange(n, device=step.device) * 0x9E3779B9 + key) & MASK
    x = ((x ^ (x >> 15)) * 0x3C6EF373) & MASK
    x = ((x ^ (x >> 13)) * 0xBB67AE85) & MASK
    return (x ^ (x >> 16)).to(torch.int64)


def rounded(x, bits, positive):
    """(e4m3 codes, scales) of x, each element rounded up with the probability of its place between two
    neighbours (20 random bits); the scale is the least power of two that keeps a block's largest in
    range. `positive`: a nonzero element never becomes zero."""
    x = x.view(-1, BLOCK)
    top = x.abs().view(torch.int32).amax(1, keepdim=True)
    e = ((top + 0x1FFFFF) >> 23).clamp(min=24)
    w = x.abs() * ((262 - e) << 23).view(torch.float32)
    bits = bits.to(torch.int32).view(-1, BLOCK)
    q = (((w.view(torch.int32) + bits) >> 20) << 20).view(torch.float32)
    low = torch.floor(w * 512 + bits.float() * 2.0 ** -20) / 512
    q = torch.where(w < 2.0 ** -6, low, q)
    if positive:
        q = torch.where((x > 0) & (q == 0), 2.0 ** -9, q)
    lost = top >= 0x7F800000
    scale = torch.where(lost, math.nan, ((e - 8) << 23).view(torch.float32))
    q = torch.where(lost, 0.0, torch.where(x < 0, -q, q))
    return q.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = 2 if case.get("dtype") == "bf16" else 4
    if case["op"] == "attention":
        lens = lengths_of(case)
        h, kv, d, dv = case["heads"], case["kv_heads"], case["dim"], case["dim_v"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        rows = sum(lens)
        b, f = rows * (h * d + kv * (d + dv) + h * dv) * size, 2 * pairs * h * (d + dv)
        if case["grad"]:
            b += rows * (h * dv + h * d + kv * (d + dv)) * size
            f += 2 * pairs * h * (3 * d + 2 * dv)
        return {"bytes": b, "flops": f}
    if case["op"] == "layer_norm":
        n = case["rows"] * case["dim"]
        return {"bytes": n * size * (4 if case["grad"] else 2) + 8 * case["dim"] * case["affine"] * (1 + case["grad"]),
                "flops": n * (20 if case["grad"] else 8)}
    n = sum(math.prod(s) for s in shapes_of(case))
    return {"bytes": n * (16 + 16 / BLOCK), "flops": n * 20}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attention":
            return exact_attention(state)
        if case["op"] == "layer_norm":
            return exact_norm(state)
        return exact_adamw(state)


def exact_attention(state):
    case, grad = state["case"], state["case"]["grad"]
    q, k, v = (state[n].detach() for n in "qkv")
    group = case["heads"] // case["kv_heads"]
    outs = [torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in ((state["dout"], q, k, v) if grad else ())]
    out = outs[0] if grad else torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device=q.device)
    ends = state["offsets"].tolist()
    for a, z in zip(ends, ends[1:]):
        for j in range(case["heads"] if z > a else 0):
            kj, vj, qj = k[a:z, j // group].double(), v[a:z, j // group].double(), q[a:z, j].double()
            s = (qj @ kj.T) / math.sqrt(case["dim"])
            if case["causal"]:
                s = torch.where(torch.ones_like(s, dtype=torch.bool).tril(), s, -math.inf)
            p = torch.softmax(s, -1)
            out[a:z, j] = p @ vj
            if grad:
                g = state["dout"][a:z, j].double()
                dp = g @ vj.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(case["dim"])
                outs[1][a:z, j] = ds @ kj
                outs[2][a:z, j // group] += ds.T @ qj
                outs[3][a:z, j // group] += p.T @ g
    return outs if grad else out


def exact_norm(state):
    case, x, w, b = state["case"], state["x"].detach().double(), state["weight"], state["bias"]
    var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
    sd = torch.sqrt(var + 1e-6)
    xh = (x - mu) / sd
    y = xh if w is None else torch.addcmul(b.double(), xh, w.double())
    if not case["grad"]:
        return y
    dy = state["dy"].double()
    g = dy if w is None else dy * w.double()
    # the projection of g off the constant vector and off xh, over the deviation
    n = x.shape[-1]
    dx = (g - g.sum(-1, keepdim=True) / n - xh * ((g * xh).sum(-1, keepdim=True) / n)) / sd
    return [y, dx] + ([] if w is None else [(dy * xh).sum(0), dy.sum(0)])


def exact_adamw(state):
    def wide(code, scale):
        return code.double() * scale.double().repeat_interleave(BLOCK)

    t = float(state["step"]) + 1
    flat = [torch.zeros(sum(state["padded"]), dtype=torch.float64, device=state["step"].device) for _ in range(2)]
    at = 0
    for p, n, m in zip(state["params"], state["sizes"], state["padded"]):
        flat[0][at:at + n], flat[1][at:at + n] = p.detach().flatten(), p.grad.flatten()
        at += m
    p, g = flat
    m = torch.lerp(g, wide(state["exp_avg"], state["exp_avg_scale"]), BETAS[0])
    v = torch.lerp(g.square(), wide(state["exp_avg_sq"], state["exp_avg_sq_scale"]), BETAS[1])
    p = p - LR * DECAY * p - LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
    new, at = [], 0
    for q, n, z in zip(state["params"], state["sizes"], state["padded"]):
        new.append(p[at:at + n].view(q.shape))
        at += z
    # the random numbers are the same integers: 32-bit products, so their low halves
    i = torch.arange(p.numel(), device=p.device) % (1 << 32)
    h = (i * 0x9E3779B9 + int(t) * 0xA54FF53B) % (1 << 32)
    for down, by in ((15, 0x3C6EF373), (13, 0xBB67AE85), (16, 1)):
        h = ((h ^ h.div(1 << down, rounding_mode="floor")) * by) % (1 << 32)
    rest = []
    for x, r, positive in ((m, h % (1 << 20), False), (v, h.div(1 << 12, rounding_mode="floor"), True)):
        top = x.abs().view(-1, BLOCK).amax(1)
        frac, exp = torch.frexp(top)  # top = frac 2^exp, frac in [0.5, 1)
        scale = torch.exp2((exp + (frac > 0.875)).clamp(min=24 - 126).double() - 9)
        w = x.abs() / scale.repeat_interleave(BLOCK)
        step = torch.exp2(torch.floor(torch.log2(w.clamp(min=2.0 ** -6))) - 3)
        q = torch.floor(w / step + r.double() / (1 << 20)) * step
        if positive:
            q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)
        rest += [q.copysign(x), scale]
    return [new, rest + [torch.full((1,), t, dtype=torch.float64, device=p.device)]]
