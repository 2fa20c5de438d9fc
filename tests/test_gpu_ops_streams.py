"""The stand-alone operators under HIP graphs, on other streams and called twice at once: every result equals the plain
eager call's bits."""
import pytest
import torch

from bidiff import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def inputs(dev, seed, grad):
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)  # noqa: E731
    B, L, H, Hkv, D, V = 2, 150, 4, 2, 64, 803
    x = {"q": rnd(B, L, 2 * H, D), "k": rnd(B, L, 2 * Hkv, D), "v": rnd(B, L, Hkv, 2 * D), "lam": torch.rand(H, generator=g, device=dev),
         "w": rnd(V, 2 * H * D) * 0.05}
    if grad:
        x = {n: t.requires_grad_(True) for n, t in x.items()}
    x["m"] = torch.arange(L, device=dev)[None] < torch.randint(1, L + 1, (B, 1), generator=g, device=dev)
    x["t"] = torch.randint(0, V, (B, L), generator=g, device=dev)
    x["ind"] = torch.rand(B, L, generator=g, device=dev) < 0.5
    x["table"] = ops.rotary_table(D, L, device=dev)
    return x


def step(x, grad):
    q, k = ops.rotary(x["q"], x["k"], x["table"])
    o = ops.differential_attention(q, k, x["v"], x["lam"], key_mask=x["m"])
    loss = ops.linear_cross_entropy(o.flatten(-2), x["w"], x["t"], x["ind"], x["m"].long())
    if not grad:
        return (o, loss)
    return (o, loss) + torch.autograd.grad(loss, [x[n] for n in ("q", "k", "v", "lam", "w")])


def same(a, b):
    return all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("grad", [False, True])
def test_two_captured_graphs_replayed_in_turn(gpu_device, grad):
    dev = gpu_device
    sets = [inputs(dev, s, grad) for s in (1, 2)]
    fresh = [[t.detach().clone() for t in (x["q"], x["t"])] for x in (inputs(dev, 11, False), inputs(dev, 12, False))]
    graphs, outs = [], []
    for x in sets:
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            for _ in range(2):
                step(x, grad)
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, grad)
        graphs.append(graph)
        outs.append(out)
    for rep in range(4):
        for i in (0, 1):
            with torch.no_grad():           # other inputs in the same places, eager work between the replays
                if rep:
                    sets[i]["q"].copy_(fresh[i][0] * (1.0 / rep))
                    sets[i]["t"].copy_(fresh[i][1].roll(rep))
            graphs[i].replay()
            got = [t.detach().clone() for t in outs[i]]
            torch.cuda.synchronize()
            want = step({n: (t.detach().clone().requires_grad_(t.requires_grad) if torch.is_tensor(t) else t) for n, t in sets[i].items()}, grad)
            assert same(got, [t.detach() for t in want]), (rep, i)
    graphs[0].replay()                      # back to back, nothing between: the two share nothing they write
    graphs[1].replay()
    both = [[t.detach().clone() for t in o] for o in outs]
    torch.cuda.synchronize()
    for i in (0, 1):
        want = step({n: (t.detach().clone().requires_grad_(t.requires_grad) if torch.is_tensor(t) else t) for n, t in sets[i].items()}, grad)
        assert same(both[i], [t.detach() for t in want])


def test_two_streams_at_once(gpu_device):
    dev = gpu_device
    sets = [inputs(dev, s, True) for s in (3, 4)]
    want = [[t.detach().clone() for t in step(x, True)] for x in sets]
    streams = [torch.cuda.Stream(device=dev) for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    for _ in range(3):
        got = []
        for s, x in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(step(x, True))
        torch.cuda.synchronize()
        assert all(same([t.detach() for t in g], w) for g, w in zip(got, want))


def test_packed_rows_under_a_graph(gpu_device):
    dev = gpu_device
    g = torch.Generator(device=dev).manual_seed(8)
    q, k, v = (torch.randn(200, h, w, generator=g, device=dev).to(BF) for h, w in ((4, 32), (4, 32), (2, 64)))
    lam = torch.rand(200, 2, generator=g, device=dev)
    cu = torch.tensor([0, 60, 60, 190], dtype=torch.int32, device=dev)
    call = lambda: ops.differential_attention(q, k, v, lam, cu_seqlens=cu, max_seqlen=130)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for ends in ([0, 60, 60, 190], [0, 1, 100, 200], [0, 0, 0, 0]):
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, call())


def test_gradients_that_are_not_asked_for(gpu_device):
    """Any subset of the operands may need a gradient: the others' are not computed into anything."""
    dev = gpu_device
    base = inputs(dev, 5, True)
    full = step(base, True)[2:]
    for i, n in enumerate(("q", "k", "v", "lam", "w")):
        x = {m: (t.detach().requires_grad_(m == n) if torch.is_tensor(t) and t.is_floating_point() and m != "table" else t) for m, t in base.items()}
        q, k = ops.rotary(x["q"], x["k"], x["table"])
        o = ops.differential_attention(q, k, x["v"], x["lam"], key_mask=x["m"])
        (only,) = torch.autograd.grad(ops.linear_cross_entropy(o.flatten(-2), x["w"], x["t"], x["ind"], x["m"].long()), (x[n],))
        assert torch.equal(only, full[i]), n


def test_second_derivatives_are_refused(gpu_device):
    x = inputs(gpu_device, 6, True)
    (g,) = torch.autograd.grad(ops.linear_cross_entropy(x["v"].flatten(-2)[..., :256], x["w"][:, :256].contiguous(), x["t"]), (x["v"],), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), (x["v"],))
