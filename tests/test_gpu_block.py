"""Norms, dense products and the balance loss as they are used: the block around a layer of
experts, and runs of them in captured graphs."""
import pytest
import torch

from mintccl_amd import dense, experts
from mintccl_amd.common import VirtualComm
from mintccl_amd.norms import Norm, join, join_grad, norm, norm_grad
from mintccl_amd.routing import balance, balance_grad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("world,options", [(1, {}), (2, {"score": "sigmoid"}), (4, {}), (8, {"score": "sigmoid", "renormalise": False})])
def test_a_block_of_experts_and_its_gradients(dev, world, options):
    """Both sides route alike (the plain one rounds the rows that decide), so the loss is off by 32-bit sums only; the rest by 8 bits."""
    for name, off in experts.block_distances(world, dev, **options).items():
        assert off < (1e-4 if name == "loss" else experts.FAR), (name, off)


def test_a_block_refuses_another_pass_kept(dev):
    s = experts.small_layer(1, dev)
    layer = experts.ExpertLayer(VirtualComm(world_size=1, device=dev), s["router"], s["up"], s["down"], 4)
    w = torch.ones(320, device=dev)
    shared = torch.zeros(64, 320, dtype=torch.bfloat16, device=dev)
    block = experts.ExpertBlock(layer, Norm(w), shared, shared.t().contiguous(), Norm(w), w)
    x = [s["tokens"][0].float()]
    with pytest.raises(ValueError):
        block.forward(x, [1])
    with pytest.raises(ValueError):
        block.backward(x, x, [w[0]], [])
    kept = []
    new, _, _ = block.forward(x, kept)
    with pytest.raises(ValueError):
        layer.backward(s["grads"], kept[0], loss_grads=[w[0]])
    # experts and shared expert alike: of rows of zeros nothing is added (0 * anything that is finite), and the stream goes on
    zero = [torch.zeros_like(x[0])]
    assert torch.equal(block.forward(zero)[0][0], zero[0]) and torch.isfinite(new[0]).all()


def whole(dev, rows, width, seed):
    """A run of all operators, forward and backward, of its own inputs: (the inputs that may be filled anew, a function that gives the results)."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    n_experts, inner = 24, 2 * width
    router, up, down = rand(n_experts, width) * width ** -0.5, (rand(inner, width) * width ** -0.5).bfloat16(), (rand(width, inner) * inner ** -0.5).bfloat16()
    bias, before, after, gate = rand(inner).bfloat16(), Norm(1 + 0.1 * rand(width)), Norm(1 + 0.1 * rand(width), 0.1 * rand(width), "layer"), rand(rows, 1)
    stream, chosen = rand(rows, width), torch.randint(0, n_experts, (rows, 4), generator=g).int().to(dev)
    offsets = torch.tensor([0, rows // 3, rows // 3, rows], dtype=torch.int32, device=dev)
    d_loss = torch.tensor(3.0, device=dev)

    def run():
        x = norm(stream, before, dtype=torch.bfloat16)
        logits = dense.product(norm(stream, before), router)
        found = balance(logits, chosen, score="sigmoid", offsets=offsets, z=0.01)
        few = balance(logits[:8], chosen[:8])
        h, u = dense.product(x, up, bias=bias, activation="gelu_tanh", keep=True)
        y = dense.product(h, down)
        new, behind = join(stream, y, gate=gate, gate_by="sigmoid", before=after)
        one = dense.product(x[:1], up, bias=bias, activation="silu")
        j = join_grad(new, behind, new, y, gate=gate, gate_by="sigmoid", before=after)
        d_u, d_bias = dense.activation_grad(dense.input_grad(j.y, down), u, "gelu_tanh")
        d_x = dense.input_grad(d_u, up)
        d_logits = balance_grad(d_loss, logits, chosen, found, score="sigmoid", offsets=offsets, z=0.01)
        d_router = dense.weight_grad(d_logits, norm(stream, before))
        n = norm_grad(d_x, stream, before)
        return [*found, *few, new, behind, one, *(t for t in j if t is not None), d_bias, dense.weight_grad(d_u, x), dense.weight_grad(j.y, h), d_router, n.x, n.weight]
    return (stream, gate), run


def test_runs_in_two_graphs_replayed_by_turns(dev):
    """Each replay of either graph, with eager runs in between, has the bits of an eager run of its inputs of that moment."""
    runs = [whole(dev, 193, 136, 5), whole(dev, 1100, 512, 6)]
    graphs, results = [], []
    for _, run in runs:
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream(dev).wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(run())
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1, 1) if turn % 2 else (1, 0):
            (stream, gate), run = runs[i]
            g = torch.Generator().manual_seed(100 * turn + i)
            stream.copy_(torch.randn(stream.shape, generator=g))
            gate.copy_(torch.randn(gate.shape, generator=g))
            want = [t.clone() for t in run()]
            runs[1 - i][1]()                                  # (other eager work, with its workspaces)
            graphs[i].replay()
            got = [t.clone() for t in results[i]]
            torch.cuda.synchronize()
            for k, (a, b) in enumerate(zip(got, want)):
                assert torch.equal(a, b), (turn, i, k)


def test_two_graphs_at_once(dev):
    """Replays of two graphs on two streams at the same time: each has its own workspaces."""
    runs = [whole(dev, 700, 256, 7), whole(dev, 700, 256, 8)]
    graphs, results, wants = [], [], []
    for _, run in runs:
        wants.append([t.clone() for t in run()])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(run())
        graphs.append(graph)
    streams = [torch.cuda.Stream(dev) for _ in runs]
    for _ in range(5):
        for side, graph in zip(streams, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for found, want in zip(results, wants):
            for k, (a, b) in enumerate(zip(found, want)):
                assert torch.equal(a, b), k
                a.zero_() if a.is_floating_point() else a.fill_(-1)


def test_results_that_share_memory(dev):
    """A result may be the stream or the residual itself, and lie beside the other rows of one buffer; else it may share no memory with what the call reads."""
    g = torch.Generator().manual_seed(9)
    rand = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    room = rand(40, 192)
    x, y, w = room[:, :64], room[:, 64:128], rand(64, 64)
    n = Norm(rand(64))
    want = dense.product(x, w, residual=y)
    for out in (room[:, 128:], torch.empty(40, 64, device=dev)):
        assert torch.equal(dense.product(x, w, residual=y, out=out), want)
    assert torch.equal(dense.product(x, w, residual=y, out=y), want) and torch.equal(y, want)
    for bad in (x, room[:, 1:65], room[:, 60:124]):
        with pytest.raises(ValueError):
            dense.product(x, w, out=bad)
    with pytest.raises(ValueError):
        dense.product(x, w, residual=y, out=room[:, 65:129])
    with pytest.raises(ValueError):
        dense.product(x[:, :64], w, out=w[:40])
    with pytest.raises(ValueError):
        dense.product(x, w, bias=w[5], out=w[:40])
    with pytest.raises(ValueError):
        join(x, y, out=y)
    with pytest.raises(ValueError):
        join(x, y, out=room[:, 32:96])
    with pytest.raises(ValueError):
        join(x[:39], y[:39], out=x[1:])                       # (the stream, a row on)
    with pytest.raises(ValueError):
        norm(x, n, out=room[:, 8:72])
    with pytest.raises(ValueError):
        norm(x, n, dtype=torch.bfloat16, out=room.view(torch.bfloat16)[:, :64])
    want = norm(x, n)
    assert torch.equal(norm(x, n, out=room[:, 128:]), want) and torch.equal(norm(x, n, out=x), want)
    both, of = join(want, y, before=n)
    s = want.clone()
    again, also = join(s, y, before=n, out=s)
    assert torch.equal(again, both) and torch.equal(also, of) and again is s


@pytest.mark.parametrize("rows,width", [(600_011, 8192), (300_011, 16384)])
def test_more_numbers_than_32_bits_count(dev, rows, width):
    """Over 2^32 numbers in an operand or a result: the last rows are what they are alone."""
    g = torch.Generator(dev).manual_seed(3)
    x = torch.empty(rows, width, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    n = Norm(torch.empty(width, device=dev).normal_(generator=g))
    tail = x[-5:].clone()
    got = norm(x, n)
    assert torch.equal(got[-5:], norm(tail, n))
    new, behind = join(x, got, gate=n.weight, before=n)
    alone = join(tail, got[-5:].clone(), gate=n.weight, before=n)
    assert torch.equal(new[-5:], alone[0]) and torch.equal(behind[-5:], alone[1])
    d = join_grad(new, behind, new, got, gate=n.weight, before=n)
    alone = join_grad(*alone, alone[0], got[-5:].clone(), gate=n.weight, before=n)
    assert torch.equal(d.stream[-5:], alone.stream) and torch.equal(d.y[-5:], alone.y)
    del d, new, behind, got
    # sums are of bf16's exact products, in 32 bits: off by a bf16 rounding, and less than 2^-24 for each of their terms
    def near(found, want, size, terms):
        return bool(((found.double() - want).abs() <= want.abs() * 2 ** -8 + size * (terms + 2) * 2 ** -24).all())
    w = torch.empty(40, width, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    z = dense.product(x, w)
    want, size = tail.double() @ w.double().t(), tail.double().abs() @ w.double().abs().t()
    assert near(z[-5:], want, size, width)
    d_x = dense.input_grad(z, w)
    of = z[-5:].double()
    assert near(d_x[-5:], of @ w.double(), of.abs() @ w.double().abs(), 40)
    del d_x
    d_w = dense.weight_grad(z, x, dtype=torch.float32)
    want, size = torch.zeros(40, width, dtype=torch.float64, device=dev), torch.zeros(40, width, dtype=torch.float64, device=dev)
    for i in range(0, rows, 20_000):
        a, b = z[i:i + 20_000].double().t().contiguous(), x[i:i + 20_000].double()
        want += a @ b
        size += a.abs() @ b.abs()
    assert near(d_w, want, size, rows)
    d_z, _ = dense.activation_grad(x, x, "silu")
    assert torch.equal(d_z[-5:], dense.activation_grad(tail, tail, "silu")[0])
