"""GPU tests of the two ways into the operators for token streams: ordinary eager calls run in native code, everything else
behind the gnop:: operators, with the same results."""
import pytest
import torch

import gnnhwc
from gnnhwc import _native, clip_gradients, rms_norm, rms_norm_quant, rotary, rotary_frequencies, tokens

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


class Declining:
    """Stands in for the native module and takes nothing."""

    def __getattr__(self, name):
        return lambda *a: NotImplemented


@pytest.fixture
def data(device):
    g = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(s, generator=g).to(device)  # noqa: E731
    return dict(x=make(6, 5, 160).bfloat16(), r=make(6, 5, 160).bfloat16(), w=make(160), dy=make(6, 5, 160).bfloat16(), ds=make(6, 5, 160).bfloat16(),
                q=make(2, 7, 4, 64).bfloat16(), k=make(2, 7, 2, 64).bfloat16(), qw=make(64), kw=make(64), gq=make(2, 7, 4, 64).bfloat16(),
                gk=make(2, 7, 2, 64).bfloat16(), p=torch.randint(0, 99, (7, 3), generator=g).to(device), f=rotary_frequencies((8, 12, 12), device=device),
                grads=[make(33), make(4, 5).bfloat16()])


def _everything(d):
    out = []
    leaf = lambda t: t.detach().clone().requires_grad_(True)  # noqa: E731
    x, r, w = leaf(d["x"]), leaf(d["r"]), leaf(d["w"])
    with torch.no_grad():
        out += [rms_norm(x), rms_norm(x, w, 1e-5), *rms_norm(x, w, residual=r, return_sum=True), rms_norm(x, None, residual=r)]
        out += [*rms_norm_quant(x, w, block=32), *rms_norm_quant(x, w, residual=r, return_sum=True, out_dtype=torch.int8)]
    y, s = rms_norm(x, w, residual=r, return_sum=True)
    out += torch.autograd.grad([y, s], [x, r, w], [d["dy"], d["ds"]])
    out += torch.autograd.grad(rms_norm(x, None), [x], d["dy"])
    out += torch.autograd.grad(rms_norm(d["x"], w, residual=r), [r], d["dy"])  # some of the inputs only
    out += torch.autograd.grad(rms_norm(d["x"], w), [w], d["dy"])
    out += torch.autograd.grad(rms_norm(d["x"], None, residual=r), [r], d["dy"])
    q, k, qw, kw = leaf(d["q"]), leaf(d["k"]), leaf(d["qw"]), leaf(d["kw"])
    with torch.no_grad():
        out += [rotary(q, None, d["p"], d["f"], (8, 12, 12)), *rotary(q, k, d["p"], d["f"], (8, 12, 12), True)]
        out += [*rotary(q, k, d["p"][:, 0], d["f"], None, True, qw, kw)]
    a, b = rotary(q, k, d["p"], d["f"], (8, 12, 12), False, qw, kw)
    out += torch.autograd.grad([a, b], [q, k, qw, kw], [d["gq"], d["gk"]])
    out += torch.autograd.grad(rotary(q, k, d["p"], d["f"], (8, 12, 12)), [q, k], [d["gq"], d["gk"]])
    out += torch.autograd.grad(rotary(q, None, d["p"], d["f"], (8, 12, 12), q_weight=qw), [q, qw], d["gq"])
    a, b = rotary(q, k, d["p"], d["f"], (8, 12, 12), False, qw, kw)
    out += torch.autograd.grad(b, [k, kw], d["gk"])  # one of the outputs only
    grads = [g.clone() for g in d["grads"]]
    elsewhere = [torch.empty_like(g, dtype=F32) for g in grads]
    out += [clip_gradients(grads, 1.0, out=elsewhere), *elsewhere, clip_gradients(grads, 0.5), *grads]
    return [t.detach() for t in out]


def test_both_ways_agree(data, monkeypatch):
    native = _everything(data)
    monkeypatch.setattr(tokens, "_native", Declining())
    general = _everything(data)
    assert len(native) == len(general)
    for i, (a, b) in enumerate(zip(native, general)):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.contiguous().view(-1).view(torch.uint8), b.contiguous().view(-1).view(torch.uint8)), i


def test_ordinary_calls_are_native(data, monkeypatch):
    """No ordinary call reaches the general form."""
    def refuse(*a, **k):
        raise AssertionError("the general form ran")

    for name in ("rms_norm", "rms_norm_bwd", "rms_norm_quant", "rotary", "rotary_bwd"):
        monkeypatch.setattr(torch.ops.gnop, name, refuse)
    monkeypatch.setattr(tokens, "_dense", refuse)
    _everything(data)
    x = data["x"].permute(2, 0, 1).contiguous().permute(1, 2, 0)  # channels apart: not ordinary
    with pytest.raises(AssertionError, match="general form"):
        rms_norm(x)


def test_versions_move_on(device):
    """A gradient that is clipped in place has changed, for autograd too."""
    for native in (True, False):
        t = torch.ones(8, device=device)
        wide = torch.ones(4, 8, device=device)
        args = [t] if native else [t, wide[:, ::2]]
        before = t._version
        clip_gradients(args, 100.0)
        assert t._version > before
        before = t._version
        clip_gradients(args, float("inf"))
        assert t._version == before


def test_operators_pass_torchs_checks(data):
    """Schemas, fake tensors, autograd registration and tracing with dynamic shapes."""
    leaf = lambda t: t.detach().clone().requires_grad_(True)  # noqa: E731
    ops, check = torch.ops.gnop, torch.library.opcheck
    x, r, w, q, k, p, f = (data[n] for n in ("x", "r", "w", "q", "k", "p", "f"))
    check(ops.rms_norm.default, (leaf(x), leaf(r), leaf(w), 1e-6, True))
    check(ops.rms_norm.default, (leaf(x), leaf(r), None, 1e-6, False))
    check(ops.rms_norm_bwd.default, (x, r, x, w, 1e-6))
    check(ops.rms_norm_quant.default, (x, r, w, 1e-6, 32, torch.int8, True))
    check(ops.rotary.default, (leaf(q), leaf(k), p, f, [8, 12, 12], True, leaf(data["qw"]), leaf(data["kw"]), 1e-6))
    check(ops.rotary.default, (leaf(q), None, p, f, [8, 12, 12], False, None, None, 1e-6))
    check(ops.rotary_bwd.default, (q, k, q, k, p, f, [8, 12, 12], True, data["qw"], data["kw"], 1e-6))


def test_images_are_native(data, monkeypatch, device):
    """Channels-last images reach the native call as the rows they are."""
    monkeypatch.setattr(torch.ops.gnop, "rms_norm", None)
    image = torch.randn(2, 160, 3, 4, device=device).to(memory_format=torch.channels_last).requires_grad_(True)
    y, s = rms_norm(image, data["w"], residual=image, return_sum=True, channel_dim=1)
    assert y.shape == image.shape and y.is_contiguous(memory_format=torch.channels_last) and torch.equal(s, image + image)
    assert torch.autograd.grad(y.sum(), image)[0].shape == image.shape


def test_saved_tensor_hooks(data):
    """Tensors offloaded to the host between forward and backward, and gradients in other layouts."""
    x, w = data["x"].detach().clone().requires_grad_(True), data["w"].detach().clone().requires_grad_(True)
    want = torch.autograd.grad(rms_norm(x, w), [x, w], data["dy"])
    with torch.autograd.graph.save_on_cpu():
        y = rms_norm(x, w)
    got = torch.autograd.grad(y, [x, w], data["dy"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    strange = data["dy"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    got = torch.autograd.grad(rms_norm(x, w), [x, w], strange)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    q = data["q"].detach().clone().requires_grad_(True)
    args = (data["p"], data["f"], (8, 12, 12))
    want = torch.autograd.grad(rotary(q, None, *args), q, data["gq"])[0]
    got = torch.autograd.grad(rotary(q, None, *args), q, data["gq"].transpose(1, 3).contiguous().transpose(1, 3))[0]
    assert torch.equal(got, want)
    # a broadcast gradient, as that of a sum
    a, = torch.autograd.grad(rms_norm(x, w).sum(), x)
    b, = torch.autograd.grad(rms_norm(x, w), x, torch.ones_like(x))
    assert torch.equal(a, b)


def test_negated_views(device):
    """Views that only stand for negated memory go through the dispatcher, which resolves them."""
    z = torch.complex(torch.randn(4, 64, device=device), torch.randn(4, 64, device=device)).conj()
    x = z.imag
    assert x.is_neg()
    assert torch.equal(rms_norm(x), rms_norm(x.clone())) and torch.equal(rms_norm(x, residual=x), rms_norm(x.clone(), residual=x.clone()))
    f, p = rotary_frequencies((4,), device=device), torch.arange(4, device=device)
    q = x.as_strided((1, 4, 8, 8), (512, x.stride(0), 8 * x.stride(1), x.stride(1)))
    assert torch.equal(rotary(q, None, p, f), rotary(q.clone(), None, p, f))


def test_modules(device):
    m = gnnhwc.RMSNorm(64).to(device).bfloat16()
    x = torch.randn(3, 64, device=device).bfloat16()
    y, s = m(x, x)
    assert torch.equal(s, x + x) and torch.equal(m(x), rms_norm(x, m.weight, m.eps))
    assert not torch.is_grad_enabled() or y.requires_grad
    with torch.autocast("cuda", dtype=BF16):
        assert m(x).dtype == BF16
    # an operator's name in the profiler, whichever way it went
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        m(x)
    assert any(e.key == "gnop::rms_norm" for e in prof.key_averages())
