"""GPU tests of rotary against its formula in float64 (tests/token_refs.py has the bounds and where they come from)."""
import ctypes
import math

import pytest
import torch

from gnnhwc import _cabi
from gnnhwc import Rotary, rotary, rotary_frequencies
from tests import token_refs as ref

pytestmark = pytest.mark.gpu
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16
EPS = 1e-6
# Angles: sine and cosine of the float32 kernel are within 2^-22 (polynomials 3e-9, a reduction exact to 2^-26 of a revolution,
# their own roundings), i.e. 4 u of a pair's size; turning adds 3 roundings.
TURN = 8


def _normal(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, dtype=F64)).to(dtype).to(device)


def _reference(t, weight, angle, near):
    """(values, scale) of the forward in float64."""
    v = t.double()
    if weight is not None:
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * weight.double()
    return ref.turn(v, angle, near), ref.pair_size(v, angle.shape[-1], near)


def _reference_bwd(d, t, weight, angle, near):
    """dt, scale, dw, scale in float64."""
    back, size = ref.turn(d.double(), -angle, near), ref.pair_size(d.double(), angle.shape[-1], near)
    if weight is None:
        return back, size, None, None
    v, w = t.double(), weight.double()
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    h, g = v * r, back * w
    dt = r * (g - h * (g * h).mean(-1, keepdim=True))
    scale = r * (size * w.abs() + h.abs() * (size * w.abs() * h.abs()).mean(-1, keepdim=True))
    return dt, scale, (back * h).sum((0, 1, 2)), (size * h.abs()).sum((0, 1, 2))


def _check(B, L, H, Kh, D, sections, near, norm, dtype, params, device, positions=None, seed=0, train=True):
    print("rotary", B, L, H, Kh, D, sections, near, norm, dtype, params, flush=True)
    A = len(sections)
    qkv = _normal((B, L, (H + 2 * Kh) * D), dtype, device, seed)
    q, k = qkv[..., :H * D].view(B, L, H, D).detach(), qkv[..., H * D:(H + Kh) * D].view(B, L, Kh, D).detach()
    if positions is None:
        g = torch.Generator().manual_seed(seed + 1)
        positions = torch.randint(0, 5000, (B, L, A), generator=g).to(device)
    f = rotary_frequencies(sections, device=device)
    qw = kw = None
    if norm:
        qw, kw = ((1 + 0.2 * _normal((D,), F64, "cpu", seed + 2 + i)).to(params).to(device).requires_grad_(True) for i in range(2))
    inputs = [t for t in (q, k, qw, kw) if t is not None]
    for t in inputs:
        t.requires_grad_(train)
    got = rotary(q, k if Kh else None, positions, f, sections, near, qw, kw if Kh else None, EPS)
    got = got if Kh else (got,)
    angle = ref.angles(positions, f, sections)
    roundings = TURN + (ref.K if norm else 0)
    sides = [(q, qw, got[0])] + ([(k, kw, got[1])] if Kh else [])
    for i, (t, w, out) in enumerate(sides):
        assert out.is_contiguous() and out.dtype == dtype
        want, scale = _reference(t.detach(), None if w is None else w.detach(), angle, near)
        ref.check(out.detach(), want, scale, "qk"[i], roundings)
    if not train:
        return
    grads = [_normal(o.shape, dtype, device, seed + 5 + i) for i, o in enumerate(got)]
    inputs = [t for t, _w, _o in sides] + [w for _t, w, _o in sides if w is not None]
    back = torch.autograd.grad(got, inputs, grads)
    for i, (t, w, _out) in enumerate(sides):
        want, scale, dw, dw_scale = _reference_bwd(grads[i], t.detach(), None if w is None else w.detach(), angle, near)
        ref.check(back[i], want, scale, "d" + "qk"[i], roundings)
        if w is not None:
            # added up per lane over tokens and heads, then over lanes and workgroups
            chain = B * L * t.shape[2] // 512 + 64 + 32
            ref.check(back[len(sides) + i], dw, dw_scale, "dw of " + "qk"[i], roundings + chain)


CASES = [
    # B, L, heads, kv_heads, D, sections
    (1, 1, 1, 1, 2, (1,)),
    (2, 3, 1, 0, 6, (2, 1)),
    (1, 7, 3, 1, 10, (1, 1, 2)),
    (3, 5, 2, 2, 40, (10, 10)),
    (2, 9, 4, 1, 64, (8, 12, 12)),
    (1, 33, 5, 5, 64, (16, 16)),
    (2, 17, 6, 2, 72, (12, 12, 12)),
    (1, 11, 3, 3, 80, (20, 20)),
    (2, 5, 7, 1, 96, (16, 16, 16)),
    (2, 19, 8, 2, 128, (16, 24, 24)),
    (1, 4, 20, 4, 128, (16, 16, 16, 16)),
    (1, 6, 3, 3, 160, (40, 40)),
    (1, 3, 2, 1, 256, (32, 48, 48)),
    # the end of the head stays as it is
    (2, 6, 3, 1, 64, (8,)),
    (1, 5, 2, 2, 80, (4, 5)),
    (1, 5, 2, 2, 128, (16, 16)),
    # an axis without pairs
    (1, 5, 2, 2, 32, (0, 8, 8)),
]


@pytest.mark.parametrize("dtype,params", [(F32, F32), (F64, F64), (F16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("B,L,H,Kh,D,sections", CASES)
def test_forward_and_backward(B, L, H, Kh, D, sections, near, dtype, params, device):
    for norm in (False, True):
        _check(B, L, H, Kh, D, sections, near, norm, dtype, params, device)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("B,L,H,Kh,D,sections", [(2, 3000, 12, 4, 64, (16, 16)), (1, 4097, 3, 1, 128, (64,)), (70, 1, 32, 8, 128, (16, 24, 24)),
                                                 (3, 1111, 1, 1, 40, (6, 7, 7))])
def test_many_tokens(B, L, H, Kh, D, sections, norm, device):
    _check(B, L, H, Kh, D, sections, True, norm, BF16, F32, device)
    _check(B, L, H, Kh, D, sections, False, norm, F32, F32, device, train=False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,sections", [(12, (5,)), (36, (18,)), (52, (7, 9, 9)), (200, (100,)), (200, (33,)), (248, (31, 62))])
def test_near_pairs_in_heads_that_lane_vectors_divide(D, sections, dtype, device):
    """Half of the head need not be whole vectors where a lane holds the pairs of one."""
    for norm in (False, True):
        _check(2, 45, 5, 3, D, sections, True, norm, dtype, F32, device)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("L", [768, 769, 1024, 1025, 2049])
def test_walks_of_the_backward(L, dtype, device):
    """Walks of one turn and more, and last turns that not every group has."""
    for near in (False, True):
        _check(1, L, 16, 16, 64, (16, 16), near, True, dtype, dtype, device)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, F32])
def test_long_positions(kind, device):
    """Angles of hundreds of thousands of radians, to 2^24: only the position and the frequency are in 32 bits."""
    p = torch.tensor([0, 1, 1000, 65535, 131071, 999999, 2 ** 24 - 1, 2 ** 24], device=device).to(kind).view(1, 8, 1)
    for dtype in (F32, F64):
        _check(1, 8, 2, 1, 64, (32,), False, False, dtype, dtype, device, positions=p)
    negative = -p if kind != F32 else -p - 0.25
    _check(1, 8, 2, 1, 64, (32,), True, True, F32, F32, device, positions=negative)


def test_gradients_against_differences(device):
    """Central differences in float64, as for the norm."""
    q, k = _normal((2, 3, 2, 12), F64, device, 1).requires_grad_(True), _normal((2, 3, 1, 12), F64, device, 2).requires_grad_(True)
    w = [(1 + 0.2 * _normal((12,), F64, device, 3 + i)).requires_grad_(True) for i in range(2)]
    p = torch.tensor([[0, 3], [1, 7], [5, 2]], device=device)
    f = rotary_frequencies((2, 3), device=device)
    for near in (False, True):
        assert torch.autograd.gradcheck(lambda q, k, a, b: rotary(q, k, p, f, (2, 3), near, a, b, 1e-3), (q, k, *w), eps=1e-5, atol=1e-7, rtol=1e-6)
        assert torch.autograd.gradcheck(lambda q, k: rotary(q, k, p, f, (2, 3), near), (q, k), eps=1e-5, atol=1e-7, rtol=1e-6)
        assert torch.autograd.gradcheck(lambda q: rotary(q, None, p, f, (2, 3), near), (q,), eps=1e-5, atol=1e-7, rtol=1e-6)


def test_layouts_and_positions(device):
    B, L, H, D = 2, 6, 3, 64
    f, sections = rotary_frequencies((16, 16), device=device), (16, 16)
    g = torch.Generator().manual_seed(3)
    p = torch.randint(0, 100, (B, L, 2), generator=g).to(device)
    q, k = _normal((B, L, H, D), BF16, device, 1), _normal((B, L, 1, D), BF16, device, 2)
    want = rotary(q, k, p, f, sections)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)  # (B, H, L, D) memory
    shifted = torch.empty(q.numel() + 1, dtype=BF16, device=device)[1:].view(q.shape).copy_(q)  # an address that no vector divides
    apart = torch.empty((*q.shape, 2), dtype=BF16, device=device)[..., 0].copy_(q)
    for name, t in (("heads first", heads_first), ("shifted", shifted), ("channels apart", apart)):
        got = rotary(t, k, p, f, sections)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), name
    expanded = k.expand(B, L, H, D)  # one head for all: every copy is turned alike
    got = rotary(q, expanded, p, f, sections)[1]
    assert torch.equal(got, want[1].expand(B, L, H, D))
    # positions: one set for all samples, its int64, float and strided forms
    one = p[:1]
    same = rotary(q, k, one.expand(B, L, 2), f, sections)[0]
    for name, t in (("(1, L, A)", one), ("(L, A)", one[0]), ("int32", one.int()), ("float", one.float()),
                    ("strided", torch.stack([one, one], -1)[..., 0])):
        assert torch.equal(rotary(q, k, t, f, sections)[0], same), name
    f1 = rotary_frequencies((32,), device=device)
    want = rotary(q, k, p[..., :1], f1)[0]
    assert torch.equal(rotary(q, k, p[..., 0], f1)[0], want) and torch.equal(rotary(q, k, p[..., 0], f1, (32,))[0], want)
    assert torch.equal(rotary(q[:1], k[:1], p[0, :, 0], f1)[0], want[:1])


def test_module(device):
    m = Rotary(64, (8, 12, 12), qk_norm=True, interleaved=True).to(device).bfloat16()
    assert m.frequencies.dtype == F32 and m.q_weight.dtype == BF16 and sorted(m.state_dict()) == ["k_weight", "q_weight"]
    q, k = _normal((1, 5, 2, 64), BF16, device, 1), _normal((1, 5, 2, 64), BF16, device, 2)
    p = torch.arange(15, device=device).view(5, 3)
    a, b = m(q, k, p)
    w = torch.ones(64, device=device, dtype=BF16)
    c, d = rotary(q, k, p, rotary_frequencies((8, 12, 12), device=device), (8, 12, 12), True, w, w)
    assert torch.equal(a, c) and torch.equal(b, d)
    # one ladder through the whole head: the first section starts it, the others go on
    f = rotary_frequencies((8, 12, 12), ladder="head")
    assert torch.allclose(f, rotary_frequencies((32,)))
    a.sum().backward()
    assert m.q_weight.grad.shape == (64,) and m.k_weight.grad is None or (m.k_weight.grad == 0).all()


def test_values_at_the_edges(device):
    """An infinity behind the turning pairs stays one; heads of zeros; NaN only in its own head."""
    f = rotary_frequencies((4,), device=device)
    q = _normal((1, 3, 4, 32), F32, device, 1)
    q[0, 1, 2, 31] = math.inf
    q[0, 0, 0] = 0
    q[0, 2, 3, 1] = math.nan
    p = torch.tensor([3, 0, 9], device=device)
    for near in (False, True):
        y = rotary(q, None, p, f, interleaved=near)
        assert y[0, 1, 2, 31] == math.inf and torch.equal(y[..., 8:31], q[..., 8:31])
        assert torch.equal(y[0, 1, :, :8], q[0, 1, :, :8])  # position zero
        assert int(y.isnan().sum()) == 2  # the pair
        w = torch.ones(32, device=device)
        z = rotary(q, None, p, f, interleaved=near, q_weight=w)
        assert (z[0, 0, 0] == 0).all() and z[0, 2, 3].isnan().all() and int(z.isnan().sum()) == 32 + 1


def test_empty(device):
    f = rotary_frequencies((4,), device=device)
    w = torch.ones(8, device=device, requires_grad=True)
    q = torch.zeros((0, 3, 2, 8), device=device, requires_grad=True)
    y = rotary(q, None, torch.zeros((3, 1), device=device), f, q_weight=w)
    dq, dw = torch.autograd.grad(y, [q, w], torch.zeros_like(y))
    assert dq.shape == q.shape and torch.equal(dw, torch.zeros(8, device=device))


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_in_place_through_the_c_abi(norm, near, device):
    """Outputs in the place of the inputs they replace, in a packed projection; and of the incoming gradients in the backward."""
    B, L, H, Kh, D = 3, 37, 5, 2, 80
    f, sections = rotary_frequencies((10, 20), device=device), (10, 20)
    p = torch.randint(0, 300, (L, 2), generator=torch.Generator().manual_seed(1)).to(device)
    packed = _normal((B, L, (H + 2 * Kh) * D), BF16, device, 2)
    w = [(1 + 0.2 * _normal((D,), F64, "cpu", 3 + i)).to(BF16).to(device).requires_grad_(True) for i in range(2)] if norm else [None, None]
    view = lambda t: (t[..., :H * D].view(B, L, H, D), t[..., H * D:(H + Kh) * D].view(B, L, Kh, D))  # noqa: E731
    q, k = (t.clone().requires_grad_(True) for t in view(packed))
    want = rotary(q, k, p, f, sections, near, *w, EPS)
    grads = _normal(q.shape, BF16, device, 5), _normal(k.shape, BF16, device, 6)
    want_back = torch.autograd.grad(want, [q, k] + [t for t in w if t is not None], grads)

    def call(**tensors):
        c = _cabi.RotaryCall()
        c.batch, c.tokens, c.heads, c.kv_heads, c.head_dim, c.axes, c.interleaved = B, L, H, Kh, D, 2, int(near)
        c.section_end[0], c.section_end[1] = 10, 30
        c.positions, c.position_type, c.frequencies, c.eps, c.dtype, c.param_dtype = p.data_ptr(), 1, f.data_ptr(), EPS, _cabi.BF16, _cabi.BF16
        c.position_stride[0], c.position_stride[1] = 0, 2
        if norm:
            c.q_weight, c.k_weight = w[0].data_ptr(), w[1].data_ptr()
        for name, t in tensors.items():
            setattr(c, name, t.data_ptr())
            if t.dim() == 4:
                setattr(c, name + "_stride", (ctypes.c_int64 * 3)(*t.stride()[:3]))
        return c

    stream = torch.cuda.current_stream().cuda_stream
    rest = packed[..., (H + Kh) * D:].clone()
    a, b = view(packed)
    _cabi.check(_cabi.lib.gnnhwc_rotary(ctypes.byref(call(q=a, k=b, q_out=a, k_out=b)), stream), "gnnhwc_rotary")
    assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(packed[..., (H + Kh) * D:], rest)
    gq, gk = (g.clone() for g in grads)
    dw = [torch.empty(D, dtype=BF16, device=device) for _ in range(2)]
    tensors = dict(q_grad=gq, k_grad=gk, q_out=gq, k_out=gk)
    if norm:
        tensors.update(q=q.detach(), k=k.detach(), q_dweight=dw[0], k_dweight=dw[1])
    c = call(**tensors)
    ws = torch.empty(_cabi.lib.gnnhwc_rotary_bwd_workspace_bytes(ctypes.byref(c)), dtype=torch.uint8, device=device)
    _cabi.check(_cabi.lib.gnnhwc_rotary_bwd(ctypes.byref(c), ws.data_ptr(), ws.numel(), stream), "gnnhwc_rotary_bwd")
    got = [gq, gk] + (dw if norm else [])
    assert all(torch.equal(x, y) for x, y in zip(got, want_back))


def test_graph_stream_and_compile(device):
    B, L, H, D = 2, 16, 4, 64
    f, sections = rotary_frequencies((16, 16), device=device), (16, 16)
    p = torch.arange(2 * L, device=device).view(L, 2)
    q, k = _normal((B, L, H, D), BF16, device, 1).requires_grad_(True), _normal((B, L, 1, D), BF16, device, 2).requires_grad_(True)
    w = [torch.ones(D, device=device).requires_grad_(True) for _ in range(2)]
    gq, gk = _normal((B, L, H, D), BF16, device, 3), _normal((B, L, 1, D), BF16, device, 4)

    def step():
        out = rotary(q, k, p, f, sections, True, *w)
        grads = torch.autograd.grad(out, [q, k, *w], [gq, gk])
        # (without their graph: its leaves' nodes belong to the stream they were made on, which a later capture must not touch)
        return (*(t.detach() for t in out), *grads)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        q.data.copy_(_normal((B, L, H, D), BF16, device, 10 + seed))
        p.add_(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step()))

    def loss(q, k):
        a, b = rotary(q, k, p, f, sections, True, *w)
        return (a * a).float().sum() + b.float().sum()

    want = torch.autograd.grad(loss(q, k), [q, k, *w])
    got = torch.autograd.grad(torch.compile(loss, backend="aot_eager", fullgraph=True)(q, k), [q, k, *w])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(device):
    f = rotary_frequencies((8, 8), device=device)
    q, k = torch.zeros((2, 3, 4, 64), device=device), torch.zeros((2, 3, 1, 64), device=device)
    p, w = torch.zeros((3, 2), device=device, dtype=torch.int32), torch.ones(64, device=device)
    odd = torch.zeros((1, 3, 1, 7), device=device)
    wide = torch.zeros((1, 3, 1, 258), device=device)
    uneven = torch.zeros((1, 3, 1, 254), device=device)
    for call, text in ((lambda: rotary(q.cpu(), None, p, f, (8, 8)), "must be a CUDA tensor"),
                       (lambda: rotary(q[0], None, p, f, (8, 8)), "shape"),
                       (lambda: rotary(q, k.half(), p, f, (8, 8)), "k must be"), (lambda: rotary(q, k[:, :2], p, f, (8, 8)), "k must be"),
                       (lambda: rotary(q, k, p, f, (8, 9)), "frequencies"), (lambda: rotary(q, k, p, f.half(), (8, 8)), "frequencies"),
                       (lambda: rotary(q, k, p[:, :1], f, (8, 8)), "positions"), (lambda: rotary(q, k, p[:2], f, (8, 8)), "positions"),
                       (lambda: rotary(q, k, p.half(), f, (8, 8)), "positions"), (lambda: rotary(q, k, p.cpu(), f, (8, 8)), "CUDA"),
                       (lambda: rotary(q, k, p, f, (8, 8), q_weight=w), "both"), (lambda: rotary(q, None, p, f, (8, 8), k_weight=w), "without k"),
                       (lambda: rotary(q, k, p, f, (8, 8), q_weight=w, k_weight=w[:8]), "64 elements"),
                       (lambda: rotary(q, k, p, f, (8, 8), q_weight=w, k_weight=w.half()), "must be"),
                       (lambda: rotary(q, k, p, f, (4, 4, 4, 2, 2)), "1 to 4"), (lambda: rotary(q, k, p, f, (20, -4)), "sections"),
                       (lambda: rotary(q.int(), None, p, f, (8, 8)), "not implemented"),
                       (lambda: rotary(odd, None, p, f[:2], (1, 1)), "even"), (lambda: rotary(wide, None, p, f, (8, 8)), "256"),
                       (lambda: rotary(uneven, None, p, f, (8, 8)), "multiple of 8"),
                       (lambda: rotary(q[..., :16], None, p, f, (8, 8)), "sections")):
        with pytest.raises(RuntimeError, match=text):
            call()
    with pytest.raises(ValueError):
        Rotary(16, (8, 8))
