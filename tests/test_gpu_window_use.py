"""GPU tests of window_attention and window_attention_cached where programs use them: in graphs, on streams, traced, with hooks,
against long caches."""
import copy

import pytest
import torch

from gnnhwc import Dropout, window_attention, window_attention_cached
from tests import window_refs as ref
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)
from tests.test_gpu_window import normal

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def leaves(dtype, device, seed, B=2, L=300, H=4, K=2, D=64, S=None):
    return [normal((B, n, h, D), dtype, device, seed + i).requires_grad_(True) for i, (n, h) in enumerate(((L, H), (S or L, K), (S or L, K)))]


def step(q, k, v, dout, window=50, sinks=3, causal=True):
    out = window_attention(q, k, v, window, sinks, causal)
    return [out.detach(), *torch.autograd.grad(out, [q, k, v], dout)]


def captured(f):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()  # (its graph is gone before the capture: torch ends a process whose captured backward meets a living eager one)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        return graph, f()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [dict(L=300), dict(B=1, L=2000, H=2, K=1), dict(B=1, L=40, S=3000, H=2, K=1)])
def test_captured_training_steps(shape, dtype, device):
    """Two graphs with workspaces of their own, replayed in turn and at once, eager work in between."""
    torch.cuda.synchronize()
    sets = [leaves(dtype, device, 10 * i, **shape) for i in range(2)]
    douts = [normal(s[0].shape, dtype, device, 5 + 10 * i) for i, s in enumerate(sets)]
    graphs = [captured(lambda s=s, d=d: step(*s, d)) for s, d in zip(sets, douts)]
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(3):
        fresh = [leaves(dtype, device, 100 * turn + 10 * i, **shape) for i in range(2)]
        wants = [step(*f, d) for f, d in zip(fresh, douts)]
        with torch.no_grad():
            for s, f in zip(sets, fresh):
                for t, u in zip(s, f):
                    t.copy_(u)
        torch.cuda.synchronize()
        for (graph, got), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, got), want in zip(graphs, wants):
            for g, w in zip(got, want):
                assert torch.equal(g, w), turn


def test_streams(device):
    """Calls on another stream than the current one's predecessor, two at a time."""
    sets = [leaves(BF16, device, 10 * i, L=1500) for i in range(2)]
    douts = [normal(s[0].shape, BF16, device, 5 + i) for i, s in enumerate(sets)]
    wants = [step(*s, d) for s, d in zip(sets, douts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, d, stream in zip(sets, douts, streams):
            with torch.cuda.stream(stream):
                got.append(step(*s, d))
        torch.cuda.synchronize()
        for g, want in zip(got, wants):
            assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_traced(dtype, device):
    q, k, v = leaves(dtype, device, 1)
    dout = normal(q.shape, dtype, device, 9)
    n = torch.tensor([300, 33], device=device)

    def f(q, k, v):
        return window_attention(q, k, v, 20, 2, True) + window_attention(q, k, v, None, 0, False, n)

    def g(q, k, v):
        return window_attention_cached(q[:, :1], k, v, n, 20, 2)

    want, got = f(q, k, v), torch.compile(f, backend="aot_eager", fullgraph=True)(q, k, v)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, [q, k, v], dout), torch.autograd.grad(want, [q, k, v], dout)):
        # the sum of two gradients may be taken in either order
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(torch.compile(g, backend="aot_eager", fullgraph=True)(q, k, v), g(q, k, v))


def test_saved_tensors_may_be_moved_and_recomputed(device):
    q, k, v = leaves(BF16, device, 1)
    dout = normal(q.shape, BF16, device, 9)
    want = step(q, k, v, dout)
    with torch.autograd.graph.save_on_cpu():
        out = window_attention(q, k, v, 50, 3, True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [q, k, v], dout), want[1:]))
    out = torch.utils.checkpoint.checkpoint(lambda *t: window_attention(*t, 50, 3, True), q, k, v, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [q, k, v], dout), want[1:]))
    out = window_attention(q, k, v, 50, 3, True)
    with torch.no_grad():
        q.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out, [k], dout)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_expanded_inputs(dtype, device):
    """One key head for all, one sample's keys for a batch, the same tensor twice: torch adds up what comes back."""
    B, L, H, D = 3, 90, 4, 64
    q, one, shared = (normal(s, dtype, device, i).requires_grad_(True) for i, s in enumerate(((B, L, H, D), (B, L, 1, D), (1, L, H, D))))
    dout = normal(q.shape, dtype, device, 7)
    for leaf, dim in ((one, 2), (shared, 0)):
        wide = leaf.expand(B, L, H, D)
        g, = torch.autograd.grad(window_attention(q, wide, wide, 11, 2), leaf, dout)
        k, v = (wide.detach().clone().requires_grad_(True) for _ in range(2))
        dk, dv = torch.autograd.grad(window_attention(q, k, v, 11, 2), [k, v], dout)
        assert torch.equal(g, (dk + dv).sum(dim, keepdim=True))
    g, = torch.autograd.grad(window_attention(q, q, q, 11, 2), q, dout)
    parts = [q.detach().clone().requires_grad_(True) for _ in range(3)]
    dq, dk, dv = torch.autograd.grad(window_attention(*parts, 11, 2), parts, dout)
    least = 3 * ref.U[dtype] * (dq.abs() + dk.abs() + dv.abs()).double()
    assert ((g.double() - (dq.double() + dk.double() + dv.double())).abs() <= least).all()


def test_only_some_gradients(device):
    """Whichever inputs ask for them."""
    q, k, v = leaves(BF16, device, 1)
    dout = normal(q.shape, BF16, device, 9)
    want = step(q, k, v, dout)[1:]
    for i in range(3):
        one = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        g, = torch.autograd.grad(window_attention(*one, 50, 3, True), one[i], dout)
        assert torch.equal(g, want[i])


@pytest.mark.parametrize("T", [1, 20, 200])
def test_a_cache_past_32_bits(T, device):
    """2^21 tokens of 16 heads of 128 channels: offsets to 2^33 bytes, past what a 32-bit count of elements holds."""
    B, S, H, K, D, window, sinks = 1, 1 << 21, 16, 16, 128, 300, 5
    g = torch.Generator(device=device).manual_seed(1)
    q = normal((B, T, H, D), BF16, device, 1)
    k, v = (torch.empty((B, S, K, D), dtype=BF16, device=device) for _ in range(2))
    for t in (k, v):
        t[:, :40].normal_(generator=g)
        t[:, -1000:].normal_(generator=g)
    for n in (S, S - 3):
        out = window_attention_cached(q, k, v, torch.tensor([n], device=device), window, sinks)
        # the sinks and the last 600 tokens, which hold every window: sinks in front count as the window's own neighbours
        kept = torch.cat([torch.arange(sinks), torch.arange(n - 600, n)]).to(device)
        place = torch.arange(n - T, n, device=device).view(1, T, 1)
        seen = (kept <= place) & ((kept < sinks) | (place - kept <= window))
        ref.check(out, ref.attention(q, k[:, kept], v[:, kept], seen, D ** -0.5)["out"], "out")


def test_a_sequence_past_32_bits(device):
    """700000 tokens of 32 heads of 128 channels, forward and backward: the last rows are as those of the end alone."""
    L, H, K, D, window, end = 700000, 32, 4, 128, 10, 300
    g = torch.Generator(device=device).manual_seed(1)
    q, k, v, dout = (torch.empty((1, L, h, D), dtype=BF16, device=device).normal_(generator=g) for h in (H, K, K, H))
    leaf = [t.requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaf, window)
    grads = torch.autograd.grad(out, leaf, dout)
    tail = [t.detach()[:, -end:].contiguous() for t in (q, k, v)]
    want = ref.attention(*tail, ref.sees(1, end, end, window, 0, False, None, False, device), D ** -0.5, dout[:, -end:].contiguous())
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        inside = slice(2 * window, None)  # (rows that the cut does not touch)
        ref.check(got[:, -end:][:, inside], tuple(t[:, inside] for t in want[name]), name)


def test_dropout_in_a_captured_and_in_a_traced_step(device):
    """The module's masks: others at each replay, the same forward and backward."""
    m = Dropout(0.5)
    x = torch.ones((64, 256), dtype=BF16, device=device).requires_grad_(True)
    r = torch.zeros_like(x)

    def f():
        y = m(x, r)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]

    graph, (y, dx) = captured(f)
    masks = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dx) and 0.4 < float((y != 0).double().mean()) < 0.6
        masks.append(y.clone())
        f()
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])
    traced = torch.compile(copy.deepcopy(m), backend="aot_eager", fullgraph=True)
    one, two = traced(x, r), traced(x, r)
    assert torch.equal(torch.autograd.grad(one, x, torch.ones_like(one))[0], one) and not torch.equal(one, two)
