"""GPU tests of window_attention against its formula in float64 (tests/window_refs.py has the bounds and where they come from)."""
import math

import pytest
import torch

from gnnhwc import window_attention
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)
from tests import window_refs as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def normal(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype).to(device)


def run(dtype, device, B, L, S, H, K, D, window, sinks, causal, lengths=None, scale=None, seed=0, gain=1.0):
    print("window_attention", dtype, B, L, S, H, K, D, window, sinks, causal, lengths, flush=True)
    q, k, v = (normal((B, n, h, D), dtype, device, seed + i, g).requires_grad_(True)
               for i, (n, h, g) in enumerate(((L, H, 1.5), (S, K, 1.0), (S, K, 1.0))))
    dout = normal((B, L, H, D), dtype, device, seed + 3, gain)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    out = window_attention(q, k, v, window, sinks, causal, n, scale)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, [q, k, v], dout)), out=out)
    seen = ref.sees(B, L, S, window, sinks, causal, n, False, device)
    want = ref.attention(q, k, v, seen, D ** -0.5 if scale is None else scale, dout)
    for name in ("out", "dq", "dk", "dv"):
        ref.check(got[name], want[name], "%s %s" % (name, dtype))
    return q, k, v, dout, n, got


# lengths around a tile's 32, 64 and 128 tokens, windows that end inside and at tiles, sinks inside and past the window
SHAPES = [
    (1, 1, 1, 1, 1, 8, None, 0, False), (2, 2, 2, 2, 1, 16, 0, 0, False), (1, 31, 31, 2, 2, 64, 3, 1, True), (2, 32, 32, 4, 2, 40, None, 0, True),
    (1, 33, 33, 3, 1, 96, 5, 2, False), (1, 63, 64, 2, 1, 128, 16, 0, False), (2, 64, 64, 1, 1, 72, 64, 4, True), (1, 65, 130, 2, 2, 64, 40, 7, True),
    (3, 127, 127, 2, 1, 24, 1, 0, False), (1, 128, 128, 6, 2, 128, 31, 33, False), (1, 129, 129, 2, 2, 80, None, 5, False),
    (2, 200, 333, 4, 1, 64, 70, 65, False), (1, 257, 257, 2, 1, 64, 128, 1, True), (1, 300, 300, 5, 5, 128, 37, 300, True),
    (1, 515, 515, 2, 1, 96, 100, 129, False), (2, 640, 640, 2, 2, 64, 63, 16, False), (1, 1030, 1030, 4, 2, 64, 200, 4, True),
    (1, 700, 1500, 2, 1, 128, None, 0, True), (1, 130, 130, 2, 1, 160, 33, 3, False), (1, 200, 200, 2, 2, 256, None, 0, True),
    (1, 70, 70, 1, 1, 248, 20, 2, False),
    # more heads than a kernel for few queries takes
    (4, 128, 128, 16, 16, 8, 0, 0, False), (4, 129, 129, 16, 16, 64, None, 0, False), (4, 200, 260, 16, 16, 64, 30, 5, True),
    (5, 150, 150, 16, 8, 128, 40, 3, False), (4, 257, 257, 16, 16, 96, 64, 33, True), (3, 140, 140, 20, 20, 160, 20, 1, False),
    (4, 130, 130, 16, 16, 256, None, 0, True), (6, 300, 300, 16, 4, 40, 10, 2, False), (5, 131, 131, 16, 16, 128, 5, 0, True),
    (9, 65, 100, 40, 20, 72, 70, 9, True),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dtype, device):
    if dtype == F32 and shape[5] > 128:
        with pytest.raises(RuntimeError, match="1 to 128"):
            run(dtype, device, *shape)
        return
    run(dtype, device, *shape)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [1, 4, 10, 66, 126, 130])
def test_heads_that_no_lane_vector_divides(D, dtype, device):
    if dtype != F32 or D <= 128:
        run(dtype, device, 2, 70, 70, 2, 1, D, 9, 2, False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lengths", [[150, 0, 1], [64, 33, 149], [200, -5, 150]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [(4, 2), (80, 40)])
def test_padded_batches(heads, lengths, causal, dtype, device):
    """Padding holds NaN: it reaches nobody, and gets zeros."""
    (H, K), B, L, D = heads, 3, 150, 64
    q, k, v, dout = (normal((B, L, h, D), dtype, device, i) for i, h in enumerate((H, K, K, H)))
    n = torch.tensor(lengths, device=device)
    seen = ref.sees(B, L, L, 21, 3, causal, n, False, device)
    want = ref.attention(q, k, v, seen, 0.2, dout)
    for t in (q, k, v, dout):
        for b, m in enumerate(lengths):
            t[b, max(0, m):] = math.nan
    for t in (q, k, v):
        t.requires_grad_(True)
    out = window_attention(q, k, v, 21, 3, causal, n, 0.2)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, [q, k, v], dout)), out=out)
    for name in ("out", "dq", "dk", "dv"):
        ref.check(got[name], want[name], name)
        for b, m in enumerate(lengths):
            assert not got[name][b, max(0, m):].any(), name


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [(2, 1), (80, 40)])
def test_values_that_are_not_finite_reach_those_that_see_them(heads, bad, causal, dtype, device):
    """One token of q, k, v or the gradient is NaN or infinite: what does not see it is as without it."""
    (H, K), B, L, D, window, sinks, at = heads, 1, 200, 64, 20, 3, 100
    seen = ref.sees(B, L, L, window, sinks, causal, None, False, device)[0]
    tensors = [normal((B, L, h, D), dtype, device, i) for i, h in enumerate((H, K, K, H))]
    want = ref.attention(*tensors[:3], seen.unsqueeze(0), D ** -0.5, tensors[3])
    by_key = seen[:, at]                         # queries that see the token
    by_query = seen[at]                          # keys that the token sees
    near = (seen[by_key].any(0))                 # keys that a query which sees it sees, too
    alone = torch.arange(L, device=device) == at
    touched = {  # tensor: rows of out, dq, dk, dv that may change
        "q": (alone, alone, by_query, by_query), "k": (by_key, by_key, near | alone, near | alone), "v": (by_key, by_key, near | alone, alone),
        "dout": (torch.zeros_like(alone), alone, by_query, by_query)}
    for i, which in enumerate(("q", "k", "v", "dout")):
        print(which, bad, causal, dtype, flush=True)
        changed = [t.clone() for t in tensors]
        changed[i][:, at, :, 5] = bad
        q, k, v = (t.requires_grad_(True) for t in changed[:3])
        out = window_attention(q, k, v, window, sinks, causal)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, [q, k, v], changed[3])), out=out)
        for name, rows in zip(("out", "dq", "dk", "dv"), touched[which]):
            ref.check(got[name][:, ~rows], tuple(t[:, ~rows] for t in want[name]), "%s with %s in %s" % (name, bad, which))
        if which == "v":
            assert not torch.isfinite(got["out"][:, by_key, :, 5]).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 150, 4, 2, 64, 100), (1, 150, 80, 80, 64, 100), (2, 900, 8, 8, 128, 800), (6, 1500, 6, 3, 64, 1450)])  # with and without shared keys
def test_padding_next_to_values_that_are_not_finite(shape, dtype, device):
    """Tokens of one tile, one NaN or infinite and others padding: those still get zeros."""
    B, L, H, K, D, n = shape
    lengths = torch.full((B,), n, device=device)
    for i, bad in enumerate((math.nan, math.inf, math.nan, math.nan)):
        tensors = [normal((B, L, h, D), dtype, device, j) for j, h in enumerate((H, K, K, H))]
        tensors[i][:, [1, n - 8]] = bad
        q, k, v = (t.requires_grad_(True) for t in tensors[:3])
        out = window_attention(q, k, v, 21, 3, False, lengths)
        for name, t in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, [q, k, v], tensors[3]))):
            assert not t[:, n:].any(), (name, i)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_training_that_has_diverged(dtype, device):
    """Where all is NaN, all of the results are, without a row by row search that would take seconds."""
    q, k, v = (torch.full((2, 700, h, 64), math.nan, dtype=dtype, device=device).requires_grad_(True) for h in (8, 4, 4))
    for window, sinks in ((None, 0), (50, 4)):
        out = window_attention(q, k, v, window, sinks)
        for t in (out, *torch.autograd.grad(out, [q, k, v], torch.full_like(out, math.nan))):
            assert t.isnan().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", [(16, 2, 2, 12, 12, 64, 1, 0, False), (16, 12, 12, 4, 2, 128, None, 0, True), (8, 300, 300, 4, 4, 80, 2, 0, True),
                                   (2, 700, 700, 4, 2, 64, 9, 2, False)])
def test_gradients_of_tokens_that_see_a_few(shape, dtype, device):
    """Each gradient has dS rounded, as an operand, and itself: sqrt(2) times the error of the last rounding alone, in the norm, and
    out that one only.  (dS is a small difference there: a result that is off by its weights' rounding would show.)  A tenth more for
    how the few roundings of a small case fall."""
    B, L, S, H, K, D, window, sinks, causal = shape
    q, k, v, dout, n, got = run(dtype, device, *shape)
    want = ref.attention(q, k, v, ref.sees(B, L, S, window, sinks, causal, None, False, device), D ** -0.5, dout)
    for name, most in (("out", 1.0), ("dq", math.sqrt(2)), ("dk", math.sqrt(2)), ("dv", math.sqrt(2))):
        value = want[name][0]
        alone = float((value.to(dtype).double() - value).norm())
        assert float((got[name].detach().double() - value).norm()) < 1.1 * most * alone, name


@pytest.mark.parametrize("gain", [2.0 ** -20, 2.0 ** 12])
def test_gradients_of_any_scale_in_half_precision(gain, device):
    """float16 gradients of a scaled or an averaged loss: dS is held relative to the largest."""
    q, k, v, dout, n, got = run(F16, device, 1, 300, 300, 2, 1, 64, None, 0, False, gain=gain, seed=5)
    assert all(torch.isfinite(t).all() for t in got.values())


def test_layouts(device):
    """Slices of a packed projection, expanded, transposed and misaligned tensors give what their contiguous copies give."""
    B, L, H, K, D = 2, 100, 4, 2, 64
    qkv = normal((B, L, (H + 2 * K) * D), BF16, device, 1)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([H * D, K * D, K * D], dim=-1))
    want = window_attention(q.contiguous(), k.contiguous(), v.contiguous(), 10, 2, True)
    assert torch.equal(window_attention(q, k, v, 10, 2, True), want)
    by_heads = tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    assert torch.equal(window_attention(*by_heads, 10, 2, True), want)
    wide = tuple(torch.zeros((B, L, t.shape[2], D + 3), dtype=BF16, device=device) for t in (q, k, v))
    odd = tuple(w[..., 1:1 + D] for w in wide)
    for o, t in zip(odd, (q, k, v)):
        o.copy_(t)
    assert torch.equal(window_attention(*odd, 10, 2, True), want)
    apart = tuple(torch.empty(t.shape[:-1] + (2 * D,), dtype=BF16, device=device)[..., ::2] for t in (q, k, v))
    for o, t in zip(apart, (q, k, v)):
        o.copy_(t)
    assert torch.equal(window_attention(*apart, 10, 2, True), want)
    one = k[:, :1].expand(B, L, K, D)
    assert torch.equal(window_attention(q, one, one, 10, 2, True), window_attention(q, one.contiguous(), one.contiguous(), 10, 2, True))
    # gradients through the slices, and an expanded gradient
    qkv.requires_grad_(True)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([H * D, K * D, K * D], dim=-1))
    g, = torch.autograd.grad(window_attention(q, k, v, 10, 2, True).sum(), qkv)
    parts = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
    each = torch.autograd.grad(window_attention(*parts, 10, 2, True), parts, torch.ones((B, L, H, D), dtype=BF16, device=device))
    assert torch.equal(g, torch.cat([t.flatten(2) for t in each], dim=-1))


def test_results_are_reproducible(device):
    q, k, v, dout, n, first = run(BF16, device, 2, 400, 400, 4, 2, 64, 50, 5, False)
    for _ in range(3):
        out = window_attention(q, k, v, 50, 5, False, n)
        again = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, [q, k, v], dout)), out=out)
        assert all(torch.equal(first[name], again[name]) for name in first)


def test_gradients_against_differences(device):
    """Central differences of a float32 call along random directions: the difference of f over h = 2^-6 is off by h^2 f''' / 6
    (about 2e-4 of |f'| here, where third derivatives are of f's size) and by 2 n u |f| / h of the sums."""
    q, k, v = (normal((1, 40, h, 16), F32, device, i) for i, h in enumerate((2, 1, 1)))
    dout = normal((1, 40, 2, 16), F32, device, 9).double()

    def f(*t):
        return float((window_attention(*t, 6, 2, False).double() * dout).sum())

    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(window_attention(*leaves, 6, 2, False), leaves, dout.float())
    h = 2.0 ** -6
    for i in range(3):
        d = normal(leaves[i].shape, F32, device, 20 + i)
        d = d / d.norm()
        up, down = [[t + s * h * d if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1)]
        assert abs((f(*up) - f(*down)) / (2 * h) - float((grads[i].double() * d).sum())) < 2e-3 * float(grads[i].norm())


def test_empty_batches(device):
    for B, L, S in ((0, 5, 5), (2, 0, 0), (2, 0, 7)):
        q, k, v = (torch.zeros((B, n, 2, 64), dtype=BF16, device=device, requires_grad=True) for n in (L, S, S))
        out = window_attention(q, k, v, 4)
        assert out.shape == q.shape
        dq, dk, dv = torch.autograd.grad(out, [q, k, v], torch.zeros_like(out))
        assert dq.shape == q.shape and dk.shape == k.shape and not dk.any() and not dv.any()


def test_the_operator(device):
    q, k, v = (normal((1, 20, h, 16), F32, device, i).requires_grad_(True) for i, h in enumerate((2, 1, 1)))
    n = torch.tensor([18], device=device)
    torch.library.opcheck(torch.ops.gnop.window_attention, (q, k, v, n, 4, 1, True, False, 0.25, True), test_utils=("test_schema", "test_faketensor"))
    with pytest.raises(RuntimeError, match="once only"):
        out = window_attention(q, k, v, 4)
        g, = torch.autograd.grad(out.sum(), q, create_graph=True)
        g.sum().backward()
