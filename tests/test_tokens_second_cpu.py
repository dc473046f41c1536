"""CPU checks, on tensors without memory: the backwards of rms_norm and rotary are differentiable in all that they depend on, and in
nothing else."""
import pytest
import torch

import gnnhwc  # noqa: F401  (registers the operators)

OPS = torch.ops.gnop


def _leaf(*shape):
    return torch.zeros(shape, device="meta", requires_grad=True)


def _reached(outputs, inputs):
    grads = torch.autograd.grad([o.sum() for o in outputs], inputs, allow_unused=True)
    assert all(g is None or g.shape == i.shape for g, i in zip(grads, inputs))
    return [g is not None for g in grads]


def test_norm():
    dy, ds, s, w = _leaf(3, 8), _leaf(3, 8), _leaf(3, 8), _leaf(8)
    dx, dw = OPS.rms_norm_bwd(dy, ds, s, w, 1e-6)
    assert _reached([dx], [dy, ds, s, w]) == [True] * 4
    dx, dw = OPS.rms_norm_bwd(dy, ds, s, w, 1e-6)
    assert _reached([dw], [dy, ds, s, w]) == [True, False, True, False]
    dx, dw = OPS.rms_norm_bwd(dy, None, s, None, 1e-6)
    assert not dw.requires_grad and _reached([dx], [dy, s]) == [True, True]
    one = _leaf(8)
    assert _reached(OPS.rms_norm_bwd(one, None, one, w, 1e-6), [one, w]) == [True, True]


@pytest.mark.parametrize("with_k", [False, True])
def test_rotary(with_k):
    gq, q, gk, k, qw, kw = _leaf(1, 5, 2, 8), _leaf(1, 5, 2, 8), _leaf(1, 5, 1, 8), _leaf(1, 5, 1, 8), _leaf(8), _leaf(8)
    p, f = torch.zeros((5, 1), device="meta"), torch.zeros(4, device="meta")
    if not with_k:
        gk = k = kw = None
    given = [t for t in (gq, gk, q, k, qw, kw) if t is not None]
    out = OPS.rotary_bwd(gq, gk, q, k, p, f, [4], True, qw, kw, 1e-6)
    assert [o.requires_grad for o in out] == [True, with_k, True, with_k]
    assert _reached([o for o in out if o.requires_grad], given) == [True] * len(given)
    out = OPS.rotary_bwd(gq, gk, None, None, p, f, [4], True, None, None, 1e-6)
    assert [o.requires_grad for o in out] == [True, with_k, False, False]
    assert _reached([o for o in out if o.requires_grad], given[:2 if with_k else 1]) == [True] * (2 if with_k else 1)
