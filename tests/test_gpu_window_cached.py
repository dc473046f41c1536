"""GPU tests of window_attention_cached, and of window_attention with few queries, against the formula in float64
(tests/window_refs.py has the bounds and where they come from)."""
import math

import pytest
import torch

from gnnhwc import window_attention, window_attention_cached
from tests import window_refs as ref
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)
from tests.test_gpu_window import normal, run

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# B, T, S, H, K, D, window, sinks, lengths: one token and several, whole groups and parts of a tile of rows, one workgroup a head and
# many, windows inside one tile and across all, requests that are empty, shorter than T, and as long as the cache
CASES = [
    (1, 1, 1, 1, 1, 8, None, 0, [1]), (3, 1, 40, 4, 2, 64, None, 0, [40, 1, 0]), (2, 1, 100, 8, 1, 128, 10, 4, [100, 33]), (2, 3, 64, 5, 1, 40, 7, 2, [64, 2]),
    (1, 1, 2000, 32, 8, 128, None, 0, [2000]), (2, 1, 5000, 6, 2, 64, 1000, 3, [5000, 31]), (4, 2, 300, 3, 3, 96, 64, 0, [300, 299, 1, 129]),
    (1, 7, 1000, 20, 4, 80, 300, 16, [999]), (2, 33, 200, 2, 2, 64, 50, 5, [200, 20]), (1, 40, 3000, 6, 2, 64, 100, 33, [2500]),
    (3, 150, 400, 4, 2, 64, 60, 8, [400, 149, 170]), (2, 1, 600, 2, 1, 256, 200, 1, [600, 77]), (1, 2, 257, 3, 1, 160, None, 0, [200]),
    (2, 1, 9000, 1, 1, 128, None, 0, [9000, 4097]),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", CASES)
def test_newest_tokens(case, dtype, device):
    """What lies behind a request's length is NaN."""
    B, T, S, H, K, D, window, sinks, lengths = case
    if dtype == F32 and D > 128:
        D = 128
    print("cached", dtype, case, flush=True)
    q, k, v = (normal((B, n, h, D), dtype, device, i) for i, (n, h) in enumerate(((T, H), (S, K), (S, K))))
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    seen = ref.sees(B, T, S, window, sinks, True, n, True, device)
    want = ref.attention(q, k, v, seen, D ** -0.5)["out"]
    for b, m in enumerate(lengths):
        k[b, m:], v[b, m:] = math.nan, math.nan
    for where in (n, n.long()):
        out = window_attention_cached(q, k, v, where, window, sinks)
        ref.check(out, want, "out")
    for b, m in enumerate(lengths):
        assert not out[b, :max(0, T - m)].any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(2, 1, 700, 4, 2, 64, 90, 3, True), (1, 5, 5000, 6, 2, 128, None, 0, False), (2, 8, 333, 4, 1, 96, 20, 40, False),
                                   (1, 30, 30, 4, 2, 64, None, 0, True)])
def test_few_queries_of_a_sequence(shape, dtype, device):
    """Their gradients, too, which read what the forward left."""
    run(dtype, device, *shape)


def test_lengths_outside_the_cache_are_clamped(device):
    q, k, v = (normal((2, n, h, 64), BF16, device, i) for i, (n, h) in enumerate(((1, 4), (90, 2), (90, 2))))
    got = window_attention_cached(q, k, v, torch.tensor([-7, 2 ** 40], device=device), 30, 2)
    want = window_attention_cached(q, k, v, torch.tensor([0, 90], device=device), 30, 2)
    assert torch.equal(got, want) and not got[0].any() and got[1].all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("S", [60, 3000])
def test_values_that_are_not_finite(S, dtype, device):
    """Behind the window: no effect.  In it: on those that see it."""
    q, k, v = (normal((2, n, h, 64), dtype, device, i) for i, (n, h) in enumerate(((2, 4), (S, 2), (S, 2))))
    n = torch.tensor([S, S - 9], device=device)
    seen = ref.sees(2, 2, S, 20, 2, True, n, True, device)
    want = ref.attention(q, k, v, seen, 0.125)["out"]
    for bad in (math.nan, math.inf, -math.inf):
        kb, vb = k.clone(), v.clone()
        hidden = ~seen.any(1)
        kb[hidden], vb[hidden] = bad, bad
        ref.check(window_attention_cached(q, kb, vb, n, 20, 2), want, "out")
        vb[0, S - 2, :, 3] = bad
        out = window_attention_cached(q, kb, vb, n, 20, 2)
        assert not torch.isfinite(out[0, :, :, 3]).any()
        ref.check(out[1], tuple(t[1] for t in want), "out")
        # the oldest token that the first query sees and the second does not
        vb = v.clone()
        vb[0, S - 2 - 20] = bad
        out = window_attention_cached(q, k, vb, n, 20, 2)
        assert not torch.isfinite(out[0, 0]).any()
        ref.check(out[0, 1], tuple(t[0, 1] for t in want), "out")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,S", [(40, 60), (40, 5000), (200, 300)])
def test_rows_in_front_of_a_short_request_are_zeros_whatever_it_holds(T, S, dtype, device):
    q, k, v = (normal((2, n, h, 64), dtype, device, i) for i, (n, h) in enumerate(((T, 2), (S, 2), (S, 2))))
    for t in (q, k, v):
        t[0] = math.nan
    out = window_attention_cached(q, k, v, torch.tensor([10, S], device=device), 20, 3)
    assert not out[0, :T - 10].any() and out[0, T - 10:].isnan().all() and torch.isfinite(out[1]).all()


def test_a_step_gives_what_the_whole_sequence_gives(device):
    """Codes one at a time against a cache that grows, and all of them at once: both round to bfloat16 what is within the bound."""
    B, S, H, K, D, window, sinks = 2, 70, 4, 2, 64, 20, 3
    q, k, v = (normal((B, S, h, D), BF16, device, i) for i, h in enumerate((H, K, K)))
    whole = ref.attention(q, k, v, ref.sees(B, S, S, window, sinks, True, None, False, device), D ** -0.5)["out"]
    cache = torch.full((2, B, S, K, D), math.nan, dtype=BF16, device=device)
    for t in range(S):
        cache[0, :, t], cache[1, :, t] = k[:, t], v[:, t]
        n = torch.full((B,), t + 1, dtype=torch.int32, device=device)
        out = window_attention_cached(q[:, t:t + 1], cache[0], cache[1], n, window, sinks)
        ref.check(out[:, 0], tuple(x[:, t] for x in whole), "token %d" % t)
    ref.check(window_attention(q, k, v, window, sinks, True), whole, "all")


def test_layouts_of_caches(device):
    """Heads in front of tokens, keys and values beside each other, a slice of a larger pool: as contiguous copies."""
    B, S, K, D = 2, 130, 2, 64
    q = normal((B, 1, 8, D), BF16, device, 1)
    pool = normal((B + 1, S + 5, 2, K, D), BF16, device, 2)
    k, v = pool[1:, 3:3 + S, 0], pool[1:, 3:3 + S, 1]
    n = torch.tensor([130, 57], dtype=torch.int32, device=device)
    want = window_attention_cached(q, k.contiguous(), v.contiguous(), n, 40, 1)
    assert torch.equal(window_attention_cached(q, k, v, n, 40, 1), want)
    k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    assert torch.equal(window_attention_cached(q, k, v, n, 40, 1), want)
    assert torch.equal(window_attention_cached(q, k, v, torch.stack([n, n], 1)[:, 0], 40, 1), want)


def test_a_captured_step_reads_lengths_and_caches_at_each_replay(device):
    B, S, H, K, D = 3, 3000, 8, 2, 128
    q, k, v = (normal((B, m, h, D), BF16, device, i) for i, (m, h) in enumerate(((1, H), (S, K), (S, K))))
    n = torch.tensor([5, 6, 7], dtype=torch.int32, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        window_attention_cached(q, k, v, n, 1000, 4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention_cached(q, k, v, n, 1000, 4)
    for lengths in ([3000, 1, 0], [77, 1500, 2999], [32, 33, 2000]):
        n.copy_(torch.tensor(lengths))
        q.copy_(normal(q.shape, BF16, device, sum(lengths)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, window_attention_cached(q, k, v, n, 1000, 4)), lengths


def test_refusals(device):
    q, k = torch.zeros((2, 1, 4, 64), device=device), torch.zeros((2, 9, 2, 64), device=device)
    n = torch.tensor([9, 9], device=device)
    leaf = q.clone().requires_grad_(True)
    for call, text in ((lambda: window_attention_cached(leaf, k, k, n), "no derivative"), (lambda: window_attention_cached(q, k, k, n[:1]), "lengths"),
                       (lambda: window_attention_cached(q, k, k, n.float()), "lengths"), (lambda: window_attention_cached(q, k, k, n.cpu()), "lengths"),
                       (lambda: window_attention_cached(q, k, k[:, :8], n), "k and v"), (lambda: window_attention_cached(q, k.half(), k, n), "one type"),
                       (lambda: window_attention_cached(q.double(), k.double(), k.double(), n), "float32"),
                       (lambda: window_attention_cached(q[:, :, :3], k, k, n), "multiple"), (lambda: window_attention_cached(q, k, k, n, -1), "window"),
                       (lambda: window_attention_cached(q, k, k, n, sinks=-1), "sinks"), (lambda: window_attention_cached(q, k, k, n, scale=0.0), "scale"),
                       (lambda: window_attention_cached(q, k, k, n, scale=math.nan), "scale"), (lambda: window_attention(k, q, q), "multiple|queries"),
                       (lambda: window_attention(k.expand(2, 9, 2, 64), k[:, :8], k[:, :8]), "queries"), (lambda: window_attention(q[0], k, k), "shape"),
                       (lambda: window_attention(*(torch.zeros((1, 1, 1, 257), device=device).half(),) * 3), "256"),
                       (lambda: window_attention(*(torch.zeros((1, 1, 1, 129), device=device),) * 3), "128")):
        with pytest.raises(RuntimeError, match=text):
            call()
    with torch.no_grad():
        assert not window_attention_cached(leaf, k, k, n).any()
