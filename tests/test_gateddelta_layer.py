"""The gated delta rule, the single step and the head norm as they are used together: the GatedDelta layer, whole sequences against single
steps and against 64 bits, and captured into graphs, on other streams."""
import pytest
import torch

from pytorch_geometric_temporal_amd import ops
from pytorch_geometric_temporal_amd.nn.recurrent import GatedDelta
from test_delta import F64, recurrence
from test_group_norm import formula


def layer(backend, seed=0, **kw):
    torch.manual_seed(seed)
    m = GatedDelta(3, 16, heads=2, **kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.3 * torch.randn_like(p))
    return m.to(backend.device)


def plain(m, X, H=None, lengths=None):
    """The layer from its parameters, in the parameters' own precision (64 bits here), autograd throughout."""
    K, h = m.key_channels, m.heads
    qkv = X @ m.linear_qkv.weight.t()
    q, k, v = qkv.split([K, K, m.out_channels], -1)
    q, k = (torch.nn.functional.normalize(t.unflatten(-1, (h, -1)), dim=-1) for t in (q, k))
    forget, write = (X @ m.linear_gates.weight.t() + m.linear_gates.bias).split([h, h], -1)
    o, S = recurrence(q, k, v.unflatten(-1, (h, -1)), -m.log_rate.exp() * torch.nn.functional.softplus(forget), torch.sigmoid(write), H, lengths)
    y = formula(o.flatten(-2).reshape(-1, m.out_channels), h, m.norm_weight, m.norm_bias, m.activation, m.eps)
    return y.view(*X.shape[:-1], m.out_channels) @ m.linear_out.weight.t() + m.linear_out.bias, S


@pytest.mark.parametrize("T,key,act,ragged", [(12, None, "silu", False), (20, 8, None, True)])
def test_layer_against_64_bits(backend, T, key, act, ragged):
    """The head norm divides by the spread of eight outputs of a head: where a head's output is small against its eps the sensitivity is
    eps ** -0.5 / .. ~ 300 roundings of the rule's result; with 2^-24 * 200 for the rule that is 4e-3 at the very worst, and 1e-4 of the whole
    tensor's norm since such rows are few."""
    m = layer(backend, key_channels=key, activation=act)
    gen = torch.Generator().manual_seed(1)
    X = torch.randn(2, T, 3, 3, generator=gen)
    w = torch.randn(2, T, 3, 16, generator=gen)
    lengths = torch.tensor([[T, 3, 0], [7, T, T]]) if ragged else None
    H = 0.3 * torch.randn(2, 3, 2, m.key_channels // 2, 8, generator=gen)
    Xd, Hd = X.to(backend.device).requires_grad_(), H.to(backend.device).requires_grad_()
    Y, S = m(Xd, Hd, lengths.to(backend.device) if ragged else None)
    names = [n for n, _ in m.named_parameters()]
    got = torch.autograd.grad((Y * w.to(backend.device)).sum() + S.sum(), [Xd, Hd] + list(m.parameters()))
    ref = GatedDelta(3, 16, heads=2, key_channels=key, activation=act)
    ref.load_state_dict({n: p.detach().cpu() for n, p in m.state_dict().items()})
    ref = ref.double()
    Xr, Hr = X.to(F64).requires_grad_(), H.to(F64).requires_grad_()
    Yr, Sr = plain(ref, Xr, Hr, lengths)
    want = torch.autograd.grad((Yr * w).sum() + Sr.sum(), [Xr, Hr] + list(ref.parameters()))
    for n, a, b in zip(["Y", "S", "X", "H"] + names, (Y, S) + got, (Yr, Sr) + want):
        assert float((a.detach().cpu().to(F64) - b.detach()).norm()) <= 1e-4 * max(float(b.detach().norm()), 1e-3), n


def test_steps_answer_what_the_sequence_answers(backend):
    m = layer(backend, seed=2)
    X = torch.randn(2, 18, 3, 3, generator=torch.Generator().manual_seed(3)).to(backend.device)
    with torch.no_grad():
        Y, S = m(X)
        head, H = m(X[:, :11])
        assert torch.allclose(head, Y[:, :11], rtol=1e-4, atol=1e-5)
        for t in range(11, 18):
            assert torch.allclose(m.step(X[:, t], H), Y[:, t], rtol=1e-4, atol=1e-5)
        assert torch.allclose(H, S, rtol=1e-4, atol=1e-5)
        start = m.initial_state(2, 3, backend.device)
        m.step(X[:, 0], start)
        assert torch.allclose(start, m(X[:, :1])[1], rtol=1e-4, atol=1e-5)


def test_layer_refusals(backend):
    with pytest.raises(ValueError, match="divide"):
        GatedDelta(3, 15, heads=4)
    m = layer(backend)
    with pytest.raises(ValueError):
        m(torch.zeros(2, 4, 3, 3, device=backend.device), torch.zeros(2, 3, 2, 8, 7, device=backend.device))


def _data(dev, seed, T=40, dtype=torch.float32):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    q, k, v = unit(r(1, T, 3, 2, 32)).to(dtype), unit(r(1, T, 3, 2, 32)).to(dtype), r(1, T, 3, 4, 16).to(dtype)
    return q, k, v, -torch.nn.functional.softplus(r(1, T, 3, 4)), torch.sigmoid(r(1, T, 3, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("T,dtype", [(40, torch.float32), (300, torch.bfloat16)])
def test_captured_graphs_answer_like_eager_calls(T, dtype):
    """Two graphs of the same operators (rule with gradients, norm, step), captured from different inputs, replayed in turns with eager
    work of the same operators between the replays: every replay has the bits of the eager call."""
    dev = torch.device("cuda:0")
    w = torch.linspace(0.5, 1.5, 64, device=dev)

    def work(leaves, state):
        o, S = ops.gated_delta_rule(*leaves)
        y = ops.group_norm_act(o.flatten(0, 2).flatten(1), 4, w, None, activation="silu")
        grads = torch.autograd.grad(y.float().square().sum() + S.square().sum(), leaves)
        with torch.no_grad():
            state.copy_(S)
            step = ops.gated_delta_step(*(x.detach()[:, 0] for x in leaves), state)
        return [o.detach(), S.detach(), y.detach(), step, state, *grads]
    sets = []
    for seed in (1, 2):
        leaves = [x.requires_grad_() for x in _data(dev, seed, T, dtype)]
        state = torch.zeros(1, 3, 4, 32, 16, device=dev)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                work(leaves, state)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = work(leaves, state)
        sets.append((leaves, state, graph, outs))
    for replay in range(4):
        for n, (leaves, state, graph, outs) in enumerate(sets):
            fresh = _data(dev, 10 * replay + n, T, dtype)
            with torch.no_grad():
                for x, y in zip(leaves, fresh):
                    x.copy_(y)
            graph.replay()
            got = [x.clone() for x in outs]
            want = work([y.clone().requires_grad_() for y in fresh], torch.zeros_like(state))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (replay, n)


@pytest.mark.gpu
def test_two_streams_at_once():
    dev = torch.device("cuda:0")
    streams = [torch.cuda.Stream() for _ in range(2)]
    data = [_data(dev, s, 300) for s in (5, 6)]
    want = [ops.gated_delta_rule(*d) for d in data]
    rows = [torch.randn(500, 64, device=dev) for _ in data]
    norms = [ops.group_norm_act(r, 4) for r in rows]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((*ops.gated_delta_rule(*data[i]), ops.group_norm_act(rows[i], 4)))
    torch.cuda.synchronize()
    for i in range(2):
        for o, S, y in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(S, want[i][1]) and torch.equal(y, norms[i])
