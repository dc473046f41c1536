"""GPU tests of attention calls that the other files leave out: padded batches with fewer queries than keys, caches without room, values
that are not finite in wide heads and where workgroups share a tile's queries, calls from two threads (tests/window_refs.py has the
bounds and where they come from)."""
import math
import threading

import pytest
import torch

from gnnhwc import window_attention, window_attention_cached
from tests import window_refs as ref
from tests.left_alone import generators_left_alone  # noqa: F401 (a fixture)
from tests.test_gpu_window import normal

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def train(q, k, v, dout, *args):
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = window_attention(q, k, v, *args)
    return dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, [q, k, v], dout)), out=out)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window,sinks,causal", [(None, 0, True), (21, 3, False), (40, 70, True)])
@pytest.mark.parametrize("shape", [(5, 20, 100, 4, 2, 64), (5, 150, 400, 4, 2, 128), (5, 200, 260, 32, 16, 64), (5, 1, 90, 4, 4, 40)])
def test_padded_batches_with_fewer_queries_than_keys(shape, window, sinks, causal, dtype, device):
    """Samples that end behind the last query, among the queries, right in front of the first, far in front of it, and at once; all behind
    a sample's end is NaN."""
    B, L, S, H, K, D = shape
    lengths = [S, S - (L + 1) // 2, S - L, (S - L) // 3, 0]
    print("padded", dtype, shape, window, sinks, causal, lengths, flush=True)
    q, k, v, dout = (normal((B, n, h, D), dtype, device, i) for i, (n, h) in enumerate(((L, H), (S, K), (S, K), (L, H))))
    n = torch.tensor(lengths, device=device)
    want = ref.attention(q, k, v, ref.sees(B, L, S, window, sinks, causal, n, False, device), D ** -0.5, dout)
    for b, m in enumerate(lengths):
        k[b, m:], v[b, m:] = math.nan, math.nan
        q[b, max(0, m - (S - L)):], dout[b, max(0, m - (S - L)):] = math.nan, math.nan
    got = train(q, k, v, dout, window, sinks, causal, n)
    for name in ("out", "dq", "dk", "dv"):
        ref.check(got[name], want[name], name)
        for b, m in enumerate(lengths):
            assert not got[name][b, max(0, m - (S - L) if name in ("out", "dq") else m):].any(), name
    assert not any(got[name][2:].any() for name in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_caches_without_room(dtype, device):
    """No request holds anything: zeros, for one token and for several."""
    for T in (1, 70):
        q, k = normal((2, T, 4, 64), dtype, device, 1), torch.empty((2, 0, 2, 64), dtype=dtype, device=device)
        out = window_attention_cached(q, k, k, torch.tensor([0, 5], device=device), 3, 1)
        assert out.shape == q.shape and not out.any()
    assert window_attention_cached(q[:, :0], k, k, torch.tensor([0, 0], device=device)).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,shape", [(F16, (200, 2, 1, 160)), (BF16, (200, 2, 1, 256)), (F16, (200, 2, 1, 256)), (BF16, (200, 60, 60, 160)), (F16, (900, 8, 2, 256)),
                                         (BF16, (900, 8, 2, 160)), (F32, (200, 2, 1, 128)), (F32, (900, 8, 2, 128)), (BF16, (900, 8, 2, 64)), (F16, (900, 8, 2, 128))])
def test_values_that_are_not_finite_in_wide_heads_and_shared_tiles(dtype, shape, causal, bad, device):
    """One token of q, k, v or the gradient is NaN or infinite: what does not see it is as without it."""
    (L, H, K, D), window, sinks, at = shape, 20, 3, 100
    seen = ref.sees(1, L, L, window, sinks, causal, None, False, device)[0]
    tensors = [normal((1, L, h, D), dtype, device, i) for i, h in enumerate((H, K, K, H))]
    want = ref.attention(*tensors[:3], seen.unsqueeze(0), D ** -0.5, tensors[3])
    by_key, by_query = seen[:, at], seen[at]  # queries that see the token, keys that it sees
    near, alone = seen[by_key].any(0), torch.arange(L, device=device) == at  # near: keys that a query which sees it sees, too
    touched = {  # tensor: rows of out, dq, dk, dv that may change
        "q": (alone, alone, by_query, by_query), "k": (by_key, by_key, near | alone, near | alone), "v": (by_key, by_key, near | alone, alone),
        "dout": (torch.zeros_like(alone), alone, by_query, by_query)}
    for i, which in enumerate(touched):
        print(which, bad, causal, dtype, shape, flush=True)
        changed = [t.clone() for t in tensors]
        changed[i][:, at, :, 5] = bad
        got = train(*changed, window, sinks, causal)
        for name, rows in zip(("out", "dq", "dk", "dv"), touched[which]):
            ref.check(got[name][:, ~rows], tuple(t[:, ~rows] for t in want[name]), "%s with %s in %s" % (name, bad, which))
        if which == "v":
            assert not torch.isfinite(got["out"][:, by_key, :, 5]).any()
        if which == "dout":
            assert not torch.isfinite(got["dv"][:, by_query, :, 5]).any() and not torch.isfinite(got["dk"][:, by_query]).all()


def test_two_threads(device):
    """Each on a stream of its own, with sizes of its own: trainings that need workspaces, and tokens against caches."""
    sets = []
    for i, (L, dtype) in enumerate(((1500, BF16), (700, F32))):
        q, k, v, dout = (normal((1, L, h, 64), dtype, device, 10 * i + j) for j, h in enumerate((4, 2, 2, 4)))
        sets.append((q, k, v, dout, torch.tensor([L], device=device)))

    def work(q, k, v, dout, n):
        got = train(*(t.detach().clone() for t in (q, k, v)), dout, 50, 3, True)
        with torch.no_grad():
            return [*(t.detach() for t in got.values()), window_attention_cached(q[:, -1:], k, v, n, 300, 2)]

    wants = [work(*s) for s in sets]
    torch.cuda.synchronize()
    faults = []

    def run(s, want):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for turn in range(20):
                    got = work(*s)
                    stream.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        except BaseException as e:
            faults.append(e)

    threads = [threading.Thread(target=run, args=pair) for pair in zip(sets, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults, faults


def test_all_nan_takes_no_search(device):
    """A row that its own q or k makes NaN is filled.  Searched row by row, each would walk its keys three times, with scalar products, on
    one wavefront: matrix instructions do 16 times as many products in that time and more, and the walk of finite values is one.  Filling
    costs one more writing of the rows.  So the bound of 8 times the finite call's time is passed by far where rows are searched."""
    def once(*tensors):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        q, k, v, dout = tensors
        torch.cuda.synchronize()
        start.record()
        out = window_attention(q, k, v)
        grads = torch.autograd.grad(out, [q, k, v], dout)
        end.record()
        end.synchronize()
        return start.elapsed_time(end), (out, *grads)

    finite = [normal((2, 3000, h, 64), BF16, device, i).requires_grad_(i < 3) for i, h in enumerate((8, 4, 4, 8))]
    nothing = [torch.full_like(t, math.nan).requires_grad_(i < 3) for i, t in enumerate(finite)]
    least = min(once(*finite)[0] for _ in range(5))
    took, results = min((once(*nothing) for _ in range(5)), key=lambda r: r[0])
    print("finite %.3f ms, NaN %.3f ms" % (least, took), flush=True)
    assert all(t.isnan().all() for t in results)
    assert took < 8 * least


@pytest.mark.parametrize("which", ["gradient", "keys"])
def test_a_walk_ends_where_all_is_nan(which, device):
    """A gradient that has overflowed next to finite q, k and v, and a NaN that all queries see: all that walks such a row adds up is NaN
    after its first 64 tokens, of 4000 here, so that walks that end there read a sixtieth of what whole ones do.  The finite call takes 0.5 ms
    and a walk to the end of a row 0.3 ms for each of 32 rows that a wavefront has, twice over, 20 ms and more."""
    q, k, v, dout = (normal((4, 4000, 8, 64), BF16, device, i) for i in range(4))
    sinks = 1
    if which == "gradient":
        dout.fill_(math.nan)
    else:
        k[:, 0] = math.nan
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def once():
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        start.record()
        out = window_attention(*leaves, 1500, sinks)
        grads = torch.autograd.grad(out, leaves, dout)
        end.record()
        end.synchronize()
        return start.elapsed_time(end), (out, *grads)

    took, (out, *grads) = min((once() for _ in range(3)), key=lambda r: r[0])
    print("%s: %.3f ms" % (which, took), flush=True)
    assert all(t.isnan().all() for t in grads) and bool(out.isnan().all()) == (which == "keys")
    assert took < 20
