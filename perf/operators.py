"""Timing cases of the sequence operators: the gated delta rule (whole sequences, with gradients, and one step at a time) and
group norm with an activation on channels-last tensors.

`own` False: the operators in plain torch operations.  `own` True: this package's kernels, called as a user calls them.
"""
import math

import torch

own = False

F32 = torch.float32
F64 = torch.float64
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # a batch of 64 twelve-step windows over 207 sensors, hidden width 64 in four heads: the forward pass of a recurrent layer,
        # q / k / v read as slices of one projection
        dict(name="rule windows f32", op="rule", batch=64, steps=12, nodes=207, k_heads=4, heads=4, key=16, value=16, type="f32",
             packed=True, start=False, ragged=False, grad=False),
        # a week of five-minute readings of every sensor, each sensor's record of its own length
        dict(name="rule week bf16", op="rule", batch=1, steps=2016, nodes=207, k_heads=2, heads=2, key=32, value=32, type="bf16",
             packed=True, start=False, ragged=True, grad=False),
        # one long sequence with few heads: nothing to spread over but the sequence itself; it continues an earlier state
        dict(name="rule long bf16", op="rule", batch=1, steps=8191, nodes=1, k_heads=4, heads=8, key=128, value=128, type="bf16",
             packed=False, start=True, ragged=False, grad=False),
        # the training pass of the windows
        dict(name="rule windows f32 train", op="rule", batch=64, steps=12, nodes=207, k_heads=4, heads=4, key=16, value=16,
             type="f32", packed=False, start=False, ragged=False, grad=True),
        # the training pass over whole days of all sensors
        dict(name="rule days f32 train", op="rule", batch=4, steps=288, nodes=207, k_heads=2, heads=2, key=32, value=32, type="f32",
             packed=False, start=True, ragged=False, grad=True),
        # the training pass over a few ragged sequences, two value heads to a key head
        dict(name="rule ragged bf16 train", op="rule", batch=4, steps=1025, nodes=1, k_heads=4, heads=8, key=64, value=64, type="bf16",
             packed=False, start=False, ragged=True, grad=True),
        # answering live: one reading of every sensor, the smallest call
        dict(name="step sensors f32", op="step", batch=1, nodes=207, k_heads=4, heads=4, key=16, value=16, type="f32"),
        # one step of four samples of a 50 000-node graph
        dict(name="step 50k nodes f32", op="step", batch=4, nodes=50000, k_heads=2, heads=2, key=16, value=16, type="f32"),
        # one step of 256 sequences with wide heads
        dict(name="step wide bf16", op="step", batch=256, nodes=1, k_heads=8, heads=16, key=128, value=128, type="bf16"),
        # one window, normalised over time, sensors and the group's channels
        dict(name="norm window f32", op="norm", batch=1, rows=12 * 207, channels=64, groups=4, act="relu", type="f32", grad=False),
        # the training pass of the same over a batch
        dict(name="norm windows f32 train", op="norm", batch=64, rows=12 * 207, channels=64, groups=8, act="silu", type="f32",
             grad=True),
        # every (sample, step, node) row by itself, a group to a head: the norm behind a layer with heads, 50 000 nodes
        dict(name="norm heads bf16 train", op="norm", batch=12 * 50000, rows=1, channels=64, groups=4, act="silu", type="bf16",
             grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rule", "rule", "rule", "step", "norm", "norm"])
    kind = rng.choice(["f32", "bf16", "f16"])
    k_heads = rng.choice([1, 2, 4])
    heads = k_heads * rng.choice([1, 1, 2, 3])
    key, value = rng.choice([8, 16, 20, 32, 48, 64, 100, 128]), rng.choice([8, 16, 20, 32, 48, 64, 100, 128])
    if op == "step":
        batch, nodes = _log(rng, 1, 256), _log(rng, 1, 20000)
        while batch * nodes * heads * key * value > 60_000_000:
            batch, nodes = -(-batch // 2), -(-nodes // 2)
        return dict(op="step", batch=batch, nodes=nodes, k_heads=k_heads, heads=heads, key=key, value=value, type=kind)
    if op == "rule":
        steps, batch, nodes = _log(rng, 1, 6000), _log(rng, 1, 64), _log(rng, 1, 400)
        grad = rng.random() < 0.5
        most = (200_000_000 if grad else 500_000_000) // (heads * key * value)
        while batch * nodes * steps > max(most, 1):
            batch, nodes, steps = -(-batch // 2), -(-nodes // 2), -(-steps * 2 // 3)
        return dict(op="rule", batch=batch, steps=steps, nodes=nodes, k_heads=k_heads, heads=heads, key=key, value=value, type=kind,
                    packed=rng.random() < 0.5 and not grad, start=rng.random() < 0.5, ragged=rng.random() < 0.5, grad=grad)
    groups = rng.choice([1, 2, 3, 4, 8, 16])
    rows = rng.choice([1, _log(rng, 8, 30000)])
    channels = groups * rng.choice([8, 12, 16, 25, 32, 64] if rows == 1 else [1, 2, 4, 6, 8, 16, 25, 32, 64])
    batch = _log(rng, 1, 64) if rows > 1 else _log(rng, 64, 500000)
    while batch * rows * channels > 30_000_000:
        batch, rows = -(-batch // 2), max(1, rows // 2)
    grad = rng.random() < 0.5
    return dict(op="norm", batch=batch, rows=rows, channels=channels, groups=groups, act="silu" if grad else rng.choice(["none", "relu", "silu"]),
                type=kind, grad=grad)


# ------------------------------------------------------------------------------------------------------ inputs

def _inputs(case, seed):
    """Every input tensor of a case, from the seed alone, by name."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "norm":
        B, S, C = case["batch"], case["rows"], case["channels"]
        # activations of a network: channels of different means and widths
        x = normal(B, S, C) * (0.5 + torch.rand(C, generator=gen, device=dev)) + normal(C)
        d = dict(x=x.to(t), weight=1 + 0.2 * normal(C), bias=0.2 * normal(C))
        if case["grad"]:
            d["dy"] = normal(B, S, C).to(t)
        return d
    B, N, Hk, H, K, V = (case[n] for n in ("batch", "nodes", "k_heads", "heads", "key", "value"))
    lead = (B, case["steps"], N) if case["op"] == "rule" else (B, N)

    def unit(*shape):                                    # queries and keys come normalised
        x = normal(*shape)
        return x / x.norm(dim=-1, keepdim=True)

    q, k, v = unit(*lead, Hk, K).to(t), unit(*lead, Hk, K).to(t), normal(*lead, H, V).to(t)
    if case.get("packed"):                               # slices of one projection's output
        whole = torch.cat([q.flatten(-2), k.flatten(-2), v.flatten(-2)], -1)
        q, k, v = (p.unflatten(-1, (h, -1)) for p, h in zip(whole.split([Hk * K, Hk * K, H * V], -1), (Hk, Hk, H)))
    # log decays: most heads remember for tens of steps, some forget at once
    g = -torch.nn.functional.softplus(2 * normal(*lead, H) - 3)
    beta = torch.sigmoid(normal(*lead, H))
    d = dict(q=q, k=k, v=v, g=g, beta=beta)
    if case["op"] == "step":
        d["state"] = 0.3 * normal(B, N, H, K, V)
        return d
    d["start"] = 0.3 * normal(B, N, H, K, V) if case["start"] else None
    d["lengths"] = None
    if case["ragged"]:
        d["lengths"] = torch.randint(0, case["steps"] + 1, (B, N), generator=gen, device=dev, dtype=torch.int32)
        d["lengths"].view(-1)[0] = case["steps"]
    if case["grad"]:
        d["do"] = normal(*lead, H, V).to(t)
        d["dstate"] = 0.1 * normal(B, N, H, K, V)
    return d


def _leaves(case):
    if case["op"] == "norm":
        return ["x", "weight", "bias"]
    return ["q", "k", "v", "g", "beta"] + (["start"] if case["start"] else [])


def prepare(case, seed):
    d = _inputs(case, seed)
    if case.get("grad"):
        for n in _leaves(case):
            d[n].requires_grad_()
    d["case"] = case
    return d


# ------------------------------------------------------------------------------------------------------ plain forms

def _inverse(a):
    """(I + a)^-1 of strictly lower triangular [.., C, C], C a power of two: blocks of 2, 4, 8, .. joined by x - x a x."""
    C = a.size(-1)
    i = torch.arange(C, device=a.device)
    x = torch.eye(C, device=a.device, dtype=a.dtype).expand_as(a)
    half = 1
    while half < C:
        join = (i[:, None] // (2 * half) == i[None, :] // (2 * half)) & (i[:, None] % (2 * half) >= half) & (i[None, :] % (2 * half) < half)
        x = x - x @ (torch.where(join, a, torch.zeros_like(a)) @ x)
        half *= 2
    return x


def _rule(q, k, v, g, beta, start, lengths):
    """The rule by chunks, in float32: products inside a chunk, the state from chunk to chunk."""
    B, T, N, Hk, K = q.shape
    H, V = v.shape[-2:]
    scale = K ** -0.5
    C = min(64, 1 << max(0, (T - 1).bit_length()))
    n = -(-T // C)
    q, k, v, g, beta = (x.float() for x in (q, k, v, g, beta))
    if lengths is not None:
        inside = (torch.arange(T, device=q.device)[None, :, None] < lengths[:, None, :])[..., None]
        g, beta = (torch.where(inside, x, torch.zeros_like(x)) for x in (g, beta))
        q, k, v = (torch.where(inside[..., None], x, torch.zeros_like(x)) for x in (q, k, v))

    def chunks(x, rep):                                  # [B, T, N, h, ..] -> [B N H, n, C, ..]
        x = x.movedim(1, 3)
        x = x.repeat_interleave(rep, 2) if rep > 1 else x
        pad = [0, 0] * (x.dim() - 4) + [0, n * C - T]
        return torch.nn.functional.pad(x, pad).reshape(B * N * H, n, C, *x.shape[4:])

    q, k, v, g, beta = chunks(q * scale, H // Hk), chunks(k, H // Hk), chunks(v, 1), chunks(g, 1), chunks(beta, 1)
    c = g.double().cumsum(-1)
    low = torch.ones(C, C, device=q.device, dtype=torch.bool).tril()
    decay = torch.where(low, c[..., :, None] - c[..., None, :], torch.full((), -math.inf, device=q.device, dtype=F64)).exp().float()
    enter, leave, whole = c.exp().float(), (c[..., -1:] - c).exp().float(), c[..., -1].exp().float()
    kt = k.transpose(-1, -2)
    x = _inverse((beta[..., None] * decay * (k @ kt)).tril(-1))
    u0, w = x @ (beta[..., None] * v), x @ ((beta * enter)[..., None] * k)
    p = decay * (q @ kt)
    qe, kl = enter[..., None] * q, (leave[..., None] * k).transpose(-1, -2)
    S = start.float().reshape(B * N * H, K, V) if start is not None else torch.zeros(B * N * H, K, V, device=q.device)
    out = []
    for j in range(n):
        u = u0[:, j] - w[:, j] @ S
        out.append(qe[:, j] @ S + p[:, j] @ u)
        S = whole[:, j, None, None] * S + kl[:, j] @ u
    o = torch.cat(out, 1)[:, :T].reshape(B, N, H, T, V).movedim(3, 1)
    return o, S.reshape(B, N, H, K, V)


def _norm(x, weight, bias, groups, act, eps=1e-5):
    B, S, C = x.shape
    y = x.reshape(B, S, groups, C // groups)
    mean = y.mean((1, 3), keepdim=True)
    y = y - mean
    y = y / torch.sqrt((y * y).mean((1, 3), keepdim=True) + eps)
    y = y.reshape(B, S, C) * weight + bias
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    return y


def run(state):
    case = state["case"]
    if own:
        from pytorch_geometric_temporal_amd import ops
    if case["op"] == "norm":
        x, w, b = state["x"], state["weight"], state["bias"]
        if own:
            y = ops.group_norm_act(x, case["groups"], w, b, activation=case["act"])
        else:
            y = _norm(x.float(), w, b, case["groups"], case["act"]).to(x.dtype)
        if not case["grad"]:
            return y
        return (y, *torch.autograd.grad(y, (x, w, b), state["dy"]))
    q, k, v, g, beta = (state[n] for n in ("q", "k", "v", "g", "beta"))
    if case["op"] == "step":
        S = state["state"]
        if own:
            o = ops.gated_delta_step(q, k, v, g, beta, S)
        else:
            rep = case["heads"] // case["k_heads"]
            qf, kf = (x.float().repeat_interleave(rep, 2) for x in (q, k))
            S *= torch.exp(g)[..., None, None]
            miss = beta[..., None] * (v.float() - (kf[..., None] * S).sum(-2))
            S += kf[..., None] * miss[..., None, :]
            o = ((qf * case["key"] ** -0.5)[..., None] * S).sum(-2).to(v.dtype)
        return o, S
    if own:
        o, S = ops.gated_delta_rule(q, k, v, g, beta, state["start"], state["lengths"])
    else:
        o, S = _rule(q, k, v, g, beta, state["start"], state["lengths"])
        o = o.to(v.dtype)
    if not case["grad"]:
        return o, S
    leaves = [state[n] for n in _leaves(case)]
    return (o, S, *torch.autograd.grad((o, S), leaves, (state["do"], state["dstate"])))


# ------------------------------------------------------------------------------------------------------ 64 bits

def _rule_exact(q, k, v, g, beta, S, lengths):
    """Step by step: the state decays, the miss between the value and what the state holds for the key is written back."""
    T, rep = q.size(1), v.size(3) // q.size(3)
    out = []
    for t in range(T):
        kt, qt = k[:, t].repeat_interleave(rep, 2), q[:, t].repeat_interleave(rep, 2)
        new = S * torch.exp(g[:, t])[..., None, None]
        held = torch.einsum("bnhk,bnhkv->bnhv", kt, new)
        new = new + kt[..., None] * (beta[:, t][..., None] * (v[:, t] - held))[..., None, :]
        o = torch.einsum("bnhk,bnhkv->bnhv", qt, new) * q.size(-1) ** -0.5
        if lengths is not None:
            live = (lengths > t)[:, :, None]
            new = torch.where(live[..., None, None], new, S)
            o = torch.where(live[..., None], o, torch.zeros_like(o))
        out.append(o)
        S = new
    return torch.stack(out, 1), S


def exact(case, seed):
    d = _inputs(case, seed)
    d = {n: x.to(F64) if torch.is_tensor(x) and x.is_floating_point() else x for n, x in d.items()}
    leaves = [d[n].requires_grad_() for n in _leaves(case)] if case.get("grad") else []
    with torch.set_grad_enabled(bool(case.get("grad"))):
        if case["op"] == "norm":
            x = d["x"].unflatten(-1, (case["groups"], -1))
            centre = x - x.mean(dim=(1, 3), keepdim=True)
            z = (centre * torch.rsqrt(centre.pow(2).mean(dim=(1, 3), keepdim=True) + 1e-5)).flatten(2) * d["weight"] + d["bias"]
            y = {"none": z, "relu": z.clamp(min=0), "silu": z * torch.sigmoid(z)}[case["act"]]
            return y if not leaves else (y.detach(), *torch.autograd.grad(y, leaves, d["dy"]))
        if case["op"] == "step":
            o, S = _rule_exact(*(d[n][:, None] for n in ("q", "k", "v", "g", "beta")), d["state"], None)
            return o[:, 0], S
        B, N, H, K, V = (case[n] for n in ("batch", "nodes", "heads", "key", "value"))
        S = d["start"] if d["start"] is not None else torch.zeros(B, N, H, K, V, dtype=F64, device=d["q"].device)
        o, S = _rule_exact(d["q"], d["k"], d["v"], d["g"], d["beta"], S, d["lengths"])
        if not leaves:
            return o, S
        return (o.detach(), S.detach(), *torch.autograd.grad((o, S), leaves, (d["do"], d["dstate"])))


# ------------------------------------------------------------------------------------------------------ work

def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        n = case["batch"] * case["rows"] * case["channels"]
        if case["grad"]:                                 # x, dy in; y, dx out
            return dict(bytes=4 * n * size + 16 * case["channels"], flops=30 * n)
        return dict(bytes=2 * n * size + 8 * case["channels"], flops=10 * n)
    B, N, Hk, H, K, V = (case[n] for n in ("batch", "nodes", "k_heads", "heads", "key", "value"))
    states, rows = B * N * H * K * V, B * N
    if case["op"] == "rule":
        rows *= case["steps"]
    if case.get("ragged"):                               # lengths are spread evenly: half of the steps are there; every output row is written
        live = rows // 2
    else:
        live = rows
    read = live * ((2 * Hk * K + H * V) * size + 2 * H * 4)
    write = rows * H * V * size
    flops = live * H * 7 * K * V                         # decay, read by the key, write, read by the query
    if case["op"] == "step":
        return dict(bytes=read + write + 8 * states, flops=flops)
    ends = 4 * states * (2 if case["start"] else 1)
    if not case["grad"]:
        return dict(bytes=read + write + ends, flops=flops)
    # both passes: the inputs and the output's gradient in, the output and the gradients out
    return dict(bytes=read + 2 * write + rows * ((2 * Hk * K + H * V) * size + 2 * H * 4) + 2 * ends, flops=3 * flops)
