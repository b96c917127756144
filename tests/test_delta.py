"""Gated delta rule: sequences, gradients and single steps against the recurrence in 64 bits.

Tolerances.  A result is compared by the norm of its error over the norm of the result.  On the way to one value stand: a dot product over
K key columns, one over the 16 steps of a chunk for each of the triangular solve, P U and the decays' exponentials, for gradients one over V
value columns as well, and per chunk four more roundings of the state.  Each step of such a chain rounds by at most 2^-24 of what it
holds, so the relative error is at most about (K + V + 4 * 16 + 4 * chunks) 2^-24 times the sensitivity of the recurrence, which is at
most 2 here (unit keys, beta < 1, decays <= 1: the state update is a contraction, the solve's rows sum to less than 2).  Outputs in a
16-bit type are rounded once more, by half of its eps at most; gradients come in float32 sums and are rounded once as well."""
import pytest
import torch

from pytorch_geometric_temporal_amd import _lib, ops

F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def tolerance(K, V, T, dtype=torch.float32):
    fp32 = 2 * (K + V + 64 + 4 * ((T + 15) // 16)) * 2.0 ** -24
    return fp32 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0)


def recurrence(q, k, v, g, beta, start=None, lengths=None, scale=None):
    B, T, N, Hk, K = q.shape
    H, V = v.shape[3:]
    S = torch.zeros(B, N, H, K, V, dtype=F64) if start is None else start
    scale = K ** -0.5 if scale is None else scale
    if lengths is not None and lengths.dim() == 1:
        lengths = lengths[:, None].expand(B, N)
    out = []
    for t in range(T):
        live = torch.ones(B, N, dtype=torch.bool) if lengths is None else lengths > t
        m = live[..., None]
        pick = lambda x: torch.where(m if x.dim() == 3 else m[..., None], x, torch.zeros_like(x))  # noqa: E731
        kt = pick(k[:, t]).repeat_interleave(H // Hk, 2)
        qt = pick(q[:, t]).repeat_interleave(H // Hk, 2)
        S = torch.exp(pick(g[:, t]))[..., None, None] * S
        u = pick(beta[:, t])[..., None] * (pick(v[:, t]) - (S * kt[..., None]).sum(-2))
        S = S + kt[..., None] * u[..., None, :]
        out.append(scale * (S * qt[..., None]).sum(-2))
    return (torch.stack(out, 1) if T else torch.zeros(B, 0, N, H, V, dtype=F64)), S


def inputs(B, T, N, Hk, H, K, V, dtype, seed=0, start=True, packed=False):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=F64)  # noqa: E731
    q, k = (torch.nn.functional.normalize(r(B, T, N, Hk, K), dim=-1).to(dtype) for _ in range(2))
    v = r(B, T, N, H, V).to(dtype)
    if packed:
        whole = torch.cat([x.flatten(3) for x in (v, k, q)], -1)
        v, k, q = (p.unflatten(-1, (h, -1)) for p, h in zip(whole.split([H * V, Hk * K, Hk * K], -1), (H, Hk, Hk)))
    g = -torch.nn.functional.softplus(2 * r(B, T, N, H) - 2).float()
    beta = torch.sigmoid(r(B, T, N, H)).float()
    d = dict(q=q, k=k, v=v, g=g, beta=beta)
    d["start"] = r(B, N, H, K, V).float() if start else None
    return d, r


def error(a, b):
    a, b = a.detach().cpu().to(F64), b.detach()
    assert a.shape == b.shape, (a.shape, b.shape)
    assert bool(torch.isfinite(a).all())
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float(a.norm())


CASES = [
    # B, T, N, Hk, H, K, V: one tile, ragged tiles, every padded width, shared heads, widths that are no multiple of four
    (1, 1, 1, 1, 1, 1, 1), (2, 12, 3, 2, 2, 16, 16), (1, 16, 5, 1, 1, 8, 4), (1, 17, 2, 1, 3, 5, 7), (1, 33, 2, 2, 2, 32, 32),
    (1, 20, 1, 1, 2, 24, 20), (1, 35, 1, 1, 1, 64, 48), (1, 18, 1, 1, 1, 33, 64), (1, 19, 1, 1, 1, 128, 128), (1, 18, 1, 1, 2, 100, 9),
    (1, 17, 1, 1, 1, 16, 100),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_forward_and_gradients(backend, case, dtype):
    B, T, N, Hk, H, K, V = case
    d, r = inputs(*case, dtype, seed=T + K, packed=T % 2 == 1)
    lengths = None
    if T > 16:
        lengths = torch.randint(0, T + 1, (B, N), generator=torch.Generator().manual_seed(T))
        lengths.view(-1)[-1] = T
    check_rule(backend, d, r, case, dtype, lengths)


def check_rule(backend, d, r, case, dtype, lengths, tol=1.0):
    B, T, N, Hk, H, K, V = case
    do, dS = r(B, T, N, H, V).to(dtype), r(B, N, H, K, V).float()
    names = [n for n in ("q", "k", "v", "g", "beta", "start") if d[n] is not None]
    ref = {n: d[n].to(F64).requires_grad_() for n in names}
    o, S = recurrence(*(ref[n] for n in names[:5]), ref.get("start"), lengths)
    want = torch.autograd.grad((o, S), [ref[n] for n in names], (do.to(F64), dS.to(F64)), allow_unused=True)
    dev = {}
    for n in names:                                       # keep the strides (slices of a projection)
        x = d[n].to(backend.device)
        if d[n].stride() != x.stride():
            x = torch.empty_strided(d[n].shape, d[n].stride(), dtype=d[n].dtype, device=backend.device).copy_(d[n])
        dev[n] = x.detach().requires_grad_()
    ln = lengths.to(backend.device) if lengths is not None else None
    go, gS = ops.gated_delta_rule(*(dev[n] for n in names[:5]), dev.get("start"), ln)
    assert go.dtype == dtype and gS.dtype == torch.float32
    assert error(go, o) <= tol * tolerance(K, V, T, dtype)
    assert error(gS, S) <= tol * tolerance(K, V, T)
    got = torch.autograd.grad((go, gS), [dev[n] for n in names], (do.to(backend.device), dS.to(backend.device)))
    for n, a, b in zip(names, got, want):
        assert a.dtype == d[n].dtype and a.shape == d[n].shape
        b = torch.zeros_like(ref[n]) if b is None else b
        t = tolerance(K, V, T, dtype if n in ("q", "k", "v") else torch.float32)
        assert error(a, b) <= 2 * tol * t, (n, error(a, b), 2 * tol * t)
    if lengths is not None:                               # nothing behind a sequence
        l2 = lengths if lengths.dim() == 2 else lengths[:, None].expand(B, N)
        behind = (torch.arange(T)[None, :, None] >= l2[:, None, :])
        for x in (go, *got[:5]):
            assert not bool(x.detach().cpu()[behind].count_nonzero())
    return go, gS, got


@pytest.mark.parametrize("case", [(1, 300, 1, 1, 2, 8, 12), (1, 411, 1, 1, 1, 20, 32), (1, 272, 1, 1, 1, 33, 40)], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("ragged", [False, True])
def test_long_sequences_run_in_segments(backend, case, ragged):
    B, T, N, Hk, H, K, V = case
    d, r = inputs(*case, torch.float32, seed=T)
    dims = _lib.DeltaDimsStruct(B, T, N, Hk, H, K, V, 0, 1.0, None)
    assert _lib.get_lib()._pgt_gated_delta_segments(dims) > 2
    check_rule(backend, d, r, case, torch.float32, torch.tensor([T - 150]) if ragged else None)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 272, 1, 1, 2, 16, 16), (2, 300, 1, 1, 1, 32, 32), (1, 275, 1, 1, 2, 64, 64), (1, 257, 1, 1, 1, 128, 128),
                                  (1, 272, 1, 1, 1, 16, 9), (1, 257, 1, 1, 1, 64, 48)],
                         ids=lambda c: "x".join(map(str, c)))
def test_segments_at_whole_widths(backend, case, dtype):
    """Every whole key width and type in segments, with value widths equal and smaller, one sequence of two ending before the last segments where there are two."""
    B, T, N, Hk, H, K, V = case
    d, r = inputs(*case, dtype, seed=T + 1)
    dims = _lib.DeltaDimsStruct(B, T, N, Hk, H, K, V, TYPES.index(dtype), 1.0, None)
    assert _lib.get_lib()._pgt_gated_delta_segments(dims) > 2
    check_rule(backend, d, r, case, dtype, torch.tensor([70, T]) if B == 2 else None)


def test_lengths_of_zero_and_one_and_outside(backend):
    case = (5, 20, 2, 1, 1, 6, 5)
    d, r = inputs(*case, torch.float32, seed=4)
    lengths = torch.tensor([0, 1, 16, 20, 7])
    check_rule(backend, d, r, case, torch.float32, lengths)
    dev = {n: x.to(backend.device) for n, x in d.items()}
    args = [dev[n] for n in ("q", "k", "v", "g", "beta", "start")]
    a = ops.gated_delta_rule(*args, torch.tensor([-3, 1, 16, 99, 7], device=backend.device))
    b = ops.gated_delta_rule(*args, lengths.to(backend.device).to(torch.int32))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(a[1][0], dev["start"][0])          # a sequence of no steps hands its state on


def test_what_stands_behind_a_sequence_is_not_looked_at(backend):
    case = (2, 21, 2, 1, 2, 6, 5)
    d, r = inputs(*case, torch.float32, seed=5)
    lengths = torch.tensor([[3, 18], [0, 21]])
    behind = torch.arange(21)[None, :, None] >= lengths[:, None, :]
    plain = check_rule(backend, d, r, case, torch.float32, lengths)
    for n, bad in (("q", float("nan")), ("k", float("inf")), ("v", float("nan")), ("g", float("inf")), ("beta", float("nan"))):
        d[n] = d[n].clone()
        d[n][behind] = bad
    _, r = inputs(*case, torch.float32, seed=5)           # the same output gradients again
    dirty = check_rule(backend, d, r, case, torch.float32, lengths)
    for x, y in zip((*plain[:2], *plain[2]), (*dirty[:2], *dirty[2])):
        assert torch.equal(x, y)


def test_a_decay_of_minus_infinity_forgets(backend):
    """g = -inf at a step starts the sequence anew there: the same as the two parts by themselves."""
    case = (1, 40, 1, 1, 1, 16, 16)
    d, r = inputs(*case, torch.float32, seed=6)
    for at in (0, 5, 16, 23, 24):
        d["g"] = d["g"].clone()
        d["g"][:, at] = -float("inf")
    check_rule(backend, d, r, case, torch.float32, None)
    args = [d[n].to(backend.device) for n in ("q", "k", "v", "g", "beta")]
    o, S = ops.gated_delta_rule(*args)
    o2, S2 = ops.gated_delta_rule(*(x[:, 24:].contiguous() for x in args))
    assert error(o[:, 24:], o2.cpu().to(F64)) <= tolerance(16, 16, 40) and error(S, S2.cpu().to(F64)) <= tolerance(16, 16, 40)


def test_strong_decays_keep_their_precision(backend):
    """Sums of the log decays run into the thousands inside a chunk; their differences must not feel it."""
    case = (1, 32, 1, 1, 1, 16, 16)
    d, r = inputs(*case, torch.float32, seed=7)
    d["g"] = torch.where(torch.arange(32).reshape(1, 32, 1, 1) % 5 == 2, torch.full_like(d["g"], -150.0), d["g"])
    check_rule(backend, d, r, case, torch.float32, None)


def test_repeated_keys_without_decay(backend):
    """Every key the same, beta 1, no decay: the triangular system at its least friendly (its powers grow like binomials)."""
    case = (1, 48, 1, 1, 1, 16, 16)
    d, r = inputs(*case, torch.float32, seed=8)
    d["k"] = d["k"][:, :1].expand_as(d["k"]).contiguous()
    d["g"], d["beta"] = torch.zeros_like(d["g"]), torch.ones_like(d["beta"])
    check_rule(backend, d, r, case, torch.float32, None)


def test_gradients_against_differences(backend):
    """Central differences of the kernel's own forward along a random direction: (f(x + h) - f(x - h)) / 2h.  f's values carry a relative
    error of about 1e-6, h = 1e-2: 1e-4 of f from rounding, and a third derivative of order one gives h^2 = 1e-4 again."""
    case = (1, 20, 1, 1, 2, 6, 5)
    d, r = inputs(*case, torch.float32, seed=9)
    names = ["q", "k", "v", "g", "beta", "start"]
    w, ws = r(1, 20, 1, 2, 5).float().to(backend.device), r(1, 1, 2, 6, 5).float().to(backend.device)
    dev = {n: d[n].to(backend.device).requires_grad_() for n in names}

    def f(x):
        o, S = ops.gated_delta_rule(*(x[n] for n in names))
        return (o.double() * w).sum() + (S.double() * ws).sum()
    grads = torch.autograd.grad(f(dev), [dev[n] for n in names])
    for n, gr in zip(names, grads):
        step = r(*d[n].shape).float().to(backend.device)
        step = step / step.norm()
        with torch.no_grad():
            hi = f({**dev, n: dev[n] + 1e-2 * step})
            lo = f({**dev, n: dev[n] - 1e-2 * step})
        slope, here = float((hi - lo) / 2e-2), float((gr.double() * step).sum())
        assert abs(slope - here) <= 4e-4 * max(1.0, float(f(dev).detach().abs()), float(gr.norm())), (n, slope, here)


def test_broadcast_inputs_sum_their_gradients(backend):
    case = (2, 18, 2, 1, 2, 6, 5)
    d, _ = inputs(*case, torch.float32, seed=13)
    names = ("q", "k", "v", "g", "beta", "start")
    dev = {n: x.to(backend.device) for n, x in d.items()}
    small = {n: dev[n][:, :1].clone().requires_grad_() if n in ("k", "g") else dev[n][:1].clone().requires_grad_() for n in names}
    spread = {n: x.expand_as(dev[n]) for n, x in small.items()}
    full = {n: x.detach().contiguous().requires_grad_() for n, x in spread.items()}
    outs = []
    for x in (spread, full):
        o, S = ops.gated_delta_rule(*(x[n] for n in names))
        outs.append((o, S, o.square().sum() + S.square().sum()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    outs[0][2].backward()
    outs[1][2].backward()
    for n in names:
        want = full[n].grad.sum(1 if n in ("k", "g") else 0, keepdim=True)
        assert error(small[n].grad, want.cpu().to(F64)) <= 2.0 ** -20, n


def test_only_some_gradients(backend):
    case = (1, 18, 2, 1, 2, 6, 5)
    d, _ = inputs(*case, torch.float32, seed=10)
    dev = {n: x.to(backend.device) for n, x in d.items()}
    dev["v"].requires_grad_()
    o, S = ops.gated_delta_rule(*(dev[n] for n in ("q", "k", "v", "g", "beta", "start")))
    a, = torch.autograd.grad(S.sum(), dev["v"], retain_graph=True)      # the output's gradient is missing
    b, = torch.autograd.grad(o.sum(), dev["v"], retain_graph=True)      # the state's gradient is missing
    c, = torch.autograd.grad(o.sum() + S.sum(), dev["v"])
    assert torch.allclose(a + b, c, rtol=1e-5, atol=1e-6)
    with torch.no_grad():
        o2, S2 = ops.gated_delta_rule(*(dev[n] for n in ("q", "k", "v", "g", "beta", "start")))
    assert torch.equal(o, o2) and torch.equal(S, S2)


def test_nothing_to_do(backend):
    for B, T, N in ((0, 3, 2), (2, 0, 3), (2, 3, 0)):
        d, _ = inputs(B, T, N, 1, 2, 6, 5, torch.float32)
        dev = {n: x.to(backend.device).requires_grad_() for n, x in d.items()}
        o, S = ops.gated_delta_rule(*(dev[n] for n in ("q", "k", "v", "g", "beta", "start")))
        assert o.shape == (B, T, N, 2, 5) and torch.equal(S, dev["start"])
        (o.sum() + S.sum()).backward()
        assert torch.equal(dev["start"].grad, torch.ones_like(dev["start"])) and dev["q"].grad.shape == dev["q"].shape


STEPS = [(1, 7, 1, 1, 1, 1), (2, 3, 2, 2, 16, 16), (1, 2, 1, 3, 5, 7), (1, 2, 1, 2, 32, 24), (1, 2, 1, 1, 64, 64), (1, 1, 1, 2, 100, 128), (1, 2, 1, 1, 128, 128),
         (1, 1, 1, 1, 128, 12), (1, 1, 1, 1, 128, 33), (1, 1, 1, 1, 16, 128), (1, 1, 1, 1, 64, 100), (3, 1, 1, 1, 128, 32), (1, 1, 1, 1, 64, 20), (1, 3, 1, 1, 128, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", STEPS, ids=lambda c: "x".join(map(str, c)))
def test_single_steps(backend, case, dtype):
    B, N, Hk, H, K, V = case
    T = 3
    d, _ = inputs(B, T, N, Hk, H, K, V, dtype, seed=K + V, packed=N % 2 == 0)
    o, S = recurrence(*(d[n].to(F64) for n in ("q", "k", "v", "g", "beta", "start")))
    dev = {n: x.to(backend.device) for n, x in d.items()}
    state = dev["start"].clone()
    for t in range(T):
        got = ops.gated_delta_step(*(dev[n][:, t] for n in ("q", "k", "v", "g", "beta")), state)
        assert got.dtype == dtype
        assert error(got, o[:, t]) <= tolerance(K, V, T, dtype)
    assert error(state, S) <= tolerance(K, V, T)


def test_steps_continue_a_sequence(backend):
    case = (2, 20, 2, 1, 2, 12, 8)
    d, _ = inputs(*case, torch.float32, seed=11)
    dev = {n: x.to(backend.device) for n, x in d.items()}
    names = ("q", "k", "v", "g", "beta")
    o, S = ops.gated_delta_rule(*(dev[n] for n in names), dev["start"])
    _, state = ops.gated_delta_rule(*(dev[n][:, :13].contiguous() for n in names), dev["start"])
    for t in range(13, 20):
        got = ops.gated_delta_step(*(dev[n][:, t] for n in names), state)
        assert error(got, o[:, t].cpu().to(F64)) <= tolerance(12, 8, 20)
    assert error(state, S.cpu().to(F64)) <= tolerance(12, 8, 20)


def test_a_step_on_a_state_that_a_graph_kept_is_noticed(backend):
    d, r = inputs(1, 3, 2, 1, 2, 8, 4, torch.float32, seed=3)
    d = {n: x.to(backend.device) for n, x in d.items()}
    k = d["k"].requires_grad_()
    _, last = ops.gated_delta_rule(d["q"], k, d["v"], d["g"], d["beta"], d["start"])
    with torch.no_grad():
        ops.gated_delta_step(d["q"][:, 0], k[:, 0], d["v"][:, 0], d["g"][:, 0], d["beta"][:, 0], d["start"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        last.sum().backward()


def test_refusals(backend):
    d, _ = inputs(1, 4, 2, 1, 2, 6, 5, torch.float32)
    good = {n: x.to(backend.device) for n, x in d.items()}
    names = ("q", "k", "v", "g", "beta")

    def rule(**change):
        x = {**good, **change}
        return ops.gated_delta_rule(*(x[n] for n in names), x["start"], x.get("lengths"))
    for change, kind in [
        (dict(v=good["v"].double()), TypeError), (dict(q=good["q"].half()), TypeError), (dict(g=good["g"].half()), TypeError),
        (dict(q=None), TypeError), (dict(v=[1.0]), TypeError), (dict(lengths=torch.tensor([1.0], device=backend.device)), TypeError),
        (dict(q=good["q"][:, :3]), ValueError), (dict(k=good["k"][..., :5]), ValueError), (dict(g=good["g"][:, :3]), ValueError),
        (dict(beta=good["beta"][..., :1]), ValueError), (dict(start=good["start"][..., :4]), ValueError), (dict(v=good["v"][:, 0]), ValueError),
        (dict(lengths=torch.tensor([1, 2], device=backend.device)), ValueError),
        (dict(q=good["q"].expand(1, 4, 2, 1, 6).repeat(1, 1, 1, 3, 1), k=good["k"].repeat(1, 1, 1, 3, 1)), ValueError),
    ]:
        with pytest.raises(kind):
            rule(**change)
    wide, _ = inputs(1, 2, 1, 1, 1, 129, 4, torch.float32, start=False)
    with pytest.raises(ValueError, match="1 .. 128"):
        ops.gated_delta_rule(*(wide[n].to(backend.device) for n in names))
    one = {n: x[:, 0] for n, x in good.items() if n != "start"}
    state = good["start"].clone()
    with pytest.raises(ValueError, match="contiguous"):
        ops.gated_delta_step(*(one[n] for n in names), state.transpose(-1, -2).contiguous().transpose(-1, -2))
    with pytest.raises(TypeError):
        ops.gated_delta_step(*(one[n] for n in names), state.half())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.gated_delta_step(*(one[n].clone().requires_grad_() for n in names), state)
    assert torch.equal(state, good["start"])


def test_a_gradient_too_wide_is_refused_before_the_forward_pass(backend):
    N = 1 << 18
    z = lambda *s: torch.zeros(1, device=backend.device).expand(*s)  # noqa: E731
    q, v, gate = z(1, 1, N, 1, 128), z(1, 1, N, 1, 1), z(1, 1, N, 1)
    with pytest.raises(ValueError, match="too many for a gradient"):
        ops.gated_delta_rule(q, q, v, gate, gate.detach().requires_grad_())


def test_bad_arguments_at_the_c_entries_return_codes(backend):
    lib = _lib.get_lib()
    D = _lib.DeltaDimsStruct
    for bad in (D(1, 4, 1, 1, 1, 0, 4, 0, 1.0, None), D(1, 4, 1, 1, 1, 4, 129, 0, 1.0, None), D(1, 4, 1, 2, 3, 4, 4, 0, 1.0, None), D(-1, 4, 1, 1, 1, 4, 4, 0, 1.0, None),
                D(1, 4, 1, 1, 1, 4, 4, 7, 1.0, None), D(1 << 20, 4, 1 << 20, 1, 1, 4, 4, 0, 1.0, None)):
        assert lib._pgt_gated_delta_segments(bad) < 0 and lib.last_error()
    ok = D(1, 4, 1, 1, 1, 4, 4, 0, 1.0, None)
    with pytest.raises(_lib.PgtError, match="null pointer"):
        lib.call("pgt_gated_delta_fwd", ok, *[None] * 12, None)
    with pytest.raises(_lib.PgtError, match="null pointer"):
        lib.call("pgt_gated_delta_bwd", ok, *[None] * 18, None)
    with pytest.raises(_lib.PgtError, match="one step"):
        lib.call("pgt_gated_delta_step", ok, *[None] * 7, None)
