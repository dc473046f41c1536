"""What gnop::window_attention_bwd is handed beside the forward's tensors is held to q's sizes before anything is launched: a shorter lse
would be read past its end."""
import pytest
import torch

from gnnhwc import attention
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)

B, L, H, D = 2, 5, 4, 16
BAD = [("lse", lambda lse, rest: (lse[:0], rest)), ("lse", lambda lse, rest: (lse[:1], rest)), ("lse", lambda lse, rest: (lse[..., :-1], rest)),
       ("lse", lambda lse, rest: (lse.transpose(1, 2), rest)), ("lse", lambda lse, rest: (lse.flatten(), rest)), ("lse", lambda lse, rest: (lse.double(), rest)),
       ("lse", lambda lse, rest: (lse.half(), rest)), ("rest", lambda lse, rest: (lse, rest[:1])),
       ("rest", lambda lse, rest: (lse, rest.float()))]
ELSEWHERE = [("lse", lambda lse, rest: (lse.to("meta"), rest)), ("rest", lambda lse, rest: (lse, rest.to("meta")))]  # (torch hands these to the meta kernel)


def _kept(device):
    q = torch.zeros((B, L, H, D), dtype=torch.bfloat16, device=device)
    return q, torch.zeros((B, H, L), device=device), torch.zeros_like(q)


@pytest.mark.parametrize("name,change", BAD + ELSEWHERE)
def test_others_are_refused(name, change):
    q, lse, rest = _kept("cpu")
    attention._check_kept(q, lse, rest, "op")
    attention._check_kept(q, lse, rest[:0], "op")
    with pytest.raises(RuntimeError, match="op: %s must be" % name):
        attention._check_kept(q, *change(lse, rest), "op")


@pytest.mark.gpu
@pytest.mark.parametrize("name,change", BAD)
def test_the_operator_refuses_them(name, change, device):
    q, lse, rest = _kept(device)
    with pytest.raises(RuntimeError, match="%s must be" % name):
        torch.ops.gnop.window_attention_bwd(q, q, q, q, q, *change(lse, rest), None, 4, 1, True, 0.25)


@pytest.mark.gpu
def test_what_was_left_with_gaps_is_read(device):
    """lse in another layout than the forward's gives the same gradients."""
    g = torch.Generator(device="cpu").manual_seed(1)
    q, k, v, dout = (torch.randn((B, L, H, D), generator=g).bfloat16().to(device) for _ in range(4))
    out, lse, rest = torch.ops.gnop.window_attention(q, k, v, None, 4, 1, True, False, 0.25, True)
    want = torch.ops.gnop.window_attention_bwd(dout, q, k, v, out, lse, rest, None, 4, 1, True, 0.25)
    apart = torch.stack([lse, lse], dim=-1)[..., 0]
    got = torch.ops.gnop.window_attention_bwd(dout, q, k, v, out, apart, rest, None, 4, 1, True, 0.25)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
