"""Group norm with an activation, channels last, against the formula in 64 bits.

Tolerances (error norm over result norm).  A statistic is a sum whose longest chain of additions is the rows a thread walks, the rows a
workgroup joins, the slices and 64 lanes: below 200 in these cases.  Each addition rounds by 2^-24 of what it holds, deviations are
taken from a value of the same channel, and these inputs' means are at most 4 of their widths: 256 * 2^-24 bounds the result, twice that
a gradient (two such sums).  silu's exp and rcp add 3e-7.  16-bit results are rounded once, by half their eps."""
import pytest
import torch

from pytorch_geometric_temporal_amd import _lib, ops

F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16, torch.float16]
FP32 = 256 * 2.0 ** -24 + 3e-7


def tolerance(dtype):
    return FP32 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0)


def formula(x, groups, w, b, act, eps=1e-5):
    shape = x.shape
    z = x.reshape(shape[0], -1, groups, shape[-1] // groups)
    z = z - z.mean((1, 3), keepdim=True)
    z = (z / torch.sqrt((z * z).mean((1, 3), keepdim=True) + eps)).reshape(shape)
    z = z * w if w is not None else z
    z = z + b if b is not None else z
    return {"relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "silu": lambda: z * torch.sigmoid(z), None: lambda: z}[act]()


def make(shape, dtype, seed, weight=True, bias=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=F64)  # noqa: E731
    C = shape[-1]
    x = (r(*shape) * (0.5 + torch.rand(C, generator=gen)) + 2 * r(C)).to(dtype)
    return x, (1 + 0.2 * r(C)).float() if weight else None, (0.2 * r(C)).float() if bias else None, r(*shape).to(dtype)


def error(a, b):
    a, b = a.detach().cpu().to(F64), b.detach()
    assert a.shape == b.shape and bool(torch.isfinite(a).all())
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float(a.norm())


CASES = [
    # shape, groups: rows by themselves (vectors of 8, 4, 2, 1; clusters of 1 .. 64 lanes and several vectors a lane; more groups than a
    # workgroup holds), samples of several rows (one and many slices, odd channels, groups across vectors, rows wider than a workgroup)
    ((7, 64), 4), ((5, 12), 3), ((9, 50), 2), ((3, 16), 16), ((4, 24), 1), ((2, 1200), 1), ((3, 4128), 2), ((2, 640), 40), ((1, 8), 1),
    ((300, 32), 2), ((3, 2050), 1), ((2, 4104), 1),
    ((2, 3, 5, 64), 4), ((1, 37, 12), 3), ((3, 2, 7), 7), ((2, 9, 50), 2), ((1, 150, 6), 1), ((2, 5, 1040), 2), ((1, 3, 2100), 3), ((4, 40, 8), 2),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[0])) + f"g{c[1]}")
def test_forward_and_gradients(backend, case, dtype):
    shape, groups = case
    seed = sum(shape) + groups
    act = [None, "relu", "silu"][seed % 3]
    x, w, b, dy = make(shape, dtype, seed, weight=seed % 4 != 0, bias=seed % 5 != 0)
    leaves = [t.to(F64).requires_grad_() if t is not None else None for t in (x, w, b)]
    y = formula(leaves[0], groups, leaves[1], leaves[2], act)
    if act == "relu":      # no value so near the corner that its side could change: |z| is at least 2^10 roundings away, or it is left out
        assert bool((formula(x.to(F64), groups, w, b, None).abs() > 2.0 ** -14).float().mean() > 0.99)
        dy = torch.where(formula(x.to(F64), groups, w, b, None).abs() > 2.0 ** -14, dy, torch.zeros_like(dy))
    wanted = [t for t in leaves if t is not None]
    want = torch.autograd.grad(y, wanted, dy.to(F64))
    dev = [t.to(backend.device).requires_grad_() if t is not None else None for t in (x, w, b)]
    got = ops.group_norm_act(dev[0], groups, dev[1], dev[2], activation=act)
    assert got.dtype == dtype and got.shape == x.shape
    assert error(got, y) <= tolerance(dtype)
    grads = torch.autograd.grad(got, [t for t in dev if t is not None], dy.to(backend.device))
    for a, bb, t in zip(grads, want, wanted):
        # groups of one or two values have a gradient that cancels to almost nothing: compare with what cancels
        size = float(bb.norm()) if shape[-1] // groups * (x.numel() // shape[0] // shape[-1]) > 8 else max(float(bb.norm()), 300 * float(dy.to(F64).norm()))
        off = float((a.detach().cpu().to(F64) - bb).norm()) / size
        assert a.shape == t.shape and off <= 2 * tolerance(a.dtype), (off, a.dtype)


def test_far_means_keep_the_variance(backend):
    """Channels whose mean is 1000 of their widths: the deviations are formed before anything is squared.  x itself holds them to 2^-24 of
    the mean only, so the inputs are the exact values here and the bound is 1000 times one rounding of a deviation's input, 2^-14."""
    gen = torch.Generator().manual_seed(3)
    for shape in ((4, 64), (2, 90, 64)):
        x = (torch.randn(*shape, generator=gen) + 1000.0).float()
        y = ops.group_norm_act(x.to(backend.device), 4)
        assert error(y, formula(x.to(F64), 4, None, None, None)) <= 2.0 ** -14


@pytest.mark.parametrize("far", [60.0, 1e4])
@pytest.mark.parametrize("row", [0, 1234])
def test_a_row_far_off_keeps_the_variance(backend, far, row):
    """A single row `far` widths off, the sample's first one among them: the variance's terms are sums of squares about means that have
    this row in them, none a difference, so the bound of the other cases holds (four rows a thread, 128 threads and eight slices a sum)."""
    x, w, b, dy = make((2, 4000, 8), torch.float32, 17)
    x[:, row] += far
    leaves = [t.to(F64).requires_grad_() for t in (x, w, b)]
    y = formula(leaves[0], 2, leaves[1], leaves[2], None)
    dev = [t.to(backend.device).requires_grad_() for t in (x, w, b)]
    got = ops.group_norm_act(dev[0], 2, dev[1], dev[2])
    assert error(got, y) <= FP32
    for a, want in zip(torch.autograd.grad(got, dev, dy.to(backend.device)), torch.autograd.grad(y, leaves, dy.to(F64))):
        assert error(a, want) <= 2 * FP32


def test_only_some_gradients(backend):
    x, w, b, dy = make((3, 5, 8), torch.float32, 1)
    for shape in ((3, 5, 8), (15, 8)):
        args = [t.to(backend.device) for t in (x.view(shape), w, b)]
        full = [t.clone().requires_grad_() for t in args]
        want = torch.autograd.grad(ops.group_norm_act(full[0], 2, full[1], full[2], activation="silu"), full, dy.view(shape).to(backend.device))
        for i in range(3):
            one = [t.clone().requires_grad_(j == i) for j, t in enumerate(args)]
            got, = torch.autograd.grad(ops.group_norm_act(one[0], 2, one[1], one[2], activation="silu"), one[i], dy.view(shape).to(backend.device))
            assert torch.equal(got, want[i])


def test_layouts_and_alignment(backend):
    x, w, b, dy = make((2, 6, 16), torch.bfloat16, 2)
    want = ops.group_norm_act(x.to(backend.device), 2, w.to(backend.device), b.to(backend.device), activation="silu")
    turned = x.permute(2, 0, 1).contiguous().to(backend.device).permute(1, 2, 0)      # another order in memory
    assert torch.equal(ops.group_norm_act(turned, 2, w.to(backend.device), b.to(backend.device), activation="silu"), want)
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=backend.device)[1:].view(x.shape).copy_(x)       # two bytes off
    assert error(ops.group_norm_act(odd, 2, w.to(backend.device), b.to(backend.device), activation="silu"), want.cpu().to(F64)) <= tolerance(torch.bfloat16)
    rows = torch.empty(x.numel() + 1, dtype=x.dtype, device=backend.device)[1:].view(12, 16).copy_(x.view(12, 16))
    assert error(ops.group_norm_act(rows, 2), formula(x.view(12, 16).to(F64), 2, None, None, None)) <= tolerance(torch.bfloat16)


def test_nan_and_infinity_stay_in_their_group(backend):
    for shape in ((2, 32), (2, 7, 32)):
        x, w, b, _ = make(shape, torch.float32, 4)
        clean = ops.group_norm_act(x.to(backend.device), 4, w.to(backend.device), b.to(backend.device))
        for bad in (float("nan"), float("inf")):
            y = x.clone()
            y.view(2, -1, 32)[1, 0, 9] = bad
            got = ops.group_norm_act(y.to(backend.device), 4, w.to(backend.device), b.to(backend.device)).view(2, -1, 32)
            keep = torch.ones(2, 1, 32, dtype=torch.bool, device=backend.device)
            keep[1, :, 8:16] = False
            keep = keep.expand_as(got)
            assert torch.equal(got[keep], clean.view(2, -1, 32)[keep]) and bool(torch.isnan(got[~keep]).all())


def test_nothing_to_do(backend):
    w = torch.ones(8, device=backend.device).requires_grad_()
    for shape in ((0, 8), (0, 3, 8), (3, 0, 8)):
        x = torch.empty(*shape, device=backend.device).requires_grad_()
        y = ops.group_norm_act(x, 2, w)
        assert y.shape == x.shape
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w))


def test_refusals(backend):
    x = torch.ones(2, 3, 8, device=backend.device)
    for args, kind in [((x.double(), 2), TypeError), ((x.int(), 2), TypeError), (([1.0], 1), TypeError), ((x, 3), ValueError), ((x, 0), ValueError),
                       ((x[0, 0], 2), ValueError), ((x, 2, torch.ones(7, device=backend.device)), ValueError), ((x, 2, torch.ones(8, device=backend.device).half()), TypeError),
                       ((x, 2, None, torch.ones(2, 4, device=backend.device)), ValueError), ((x, 2, None, None, -1.0), ValueError),
                       ((x, 2, None, None, 1e-5, "gelu"), ValueError)]:
        with pytest.raises(kind):
            ops.group_norm_act(*args)
    lib = _lib.get_lib()
    assert lib._pgt_group_norm_ws_floats(2, 3, 8, 3, 0, 0) < 0 and lib.last_error()
    with pytest.raises(_lib.PgtError, match="null pointer"):
        lib.call("pgt_group_norm_act", None, 2, 3, 8, 2, 0, None, None, 1e-5, 0, None, None, None, 0, None)
    with pytest.raises(_lib.PgtError, match="ws of"):
        lib.call("pgt_group_norm_act", x.data_ptr(), 2, 3, 8, 2, 0, None, None, 1e-5, 0, x.data_ptr(), None, None, 0, None)
